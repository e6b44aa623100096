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
// that an average that moves by less than half a code per step would never move.  The draw has 16 bits, so the
// expected value is off by up to 2^-16 of the gap between the two neighbours.  A positive v never gets code 0, or the
// next update could divide a moment by eps alone: where its root is below one code it is always stored as one, larger
// than it is.  A block with a moment that is not finite is stored as NaN.
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
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// Resident CTAs per SM: at most 96 registers per thread with 8-bit moments (202M parameters: 611 us; 4 CTAs 624, 6 CTAs,
// which spill, 692), 64 with fp32 ones (184 small tensors: 18 us; 25 at 6 CTAs).
template <bool I8> constexpr int kStepCtas = I8 ? 5 : 8;
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
    uint32_t index_vec;   // index << 1 | (8 values of w and g can be accessed at once)
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
    float minus_zero;
    uint32_t plain_low, plain_high;   // v's bits for which the fast root and quotient are the IEEE ones (v in [low, high))
    uint32_t zero_is_plain;   // so they are for v = 0
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

// 32 bytes, on a 32-byte boundary, in one access: a warp's accesses then cover whole sectors, which pairs of 16-byte
// accesses at a stride of 32 do not (stores of half sectors took the read-out of 8-bit moments from 5.6 to 4.3 TB/s).
__device__ __forceinline__ void load8(const float* p, float (&x)[8])
{
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                 : "l"(__cvta_generic_to_global(p)) : "memory");
}

__device__ __forceinline__ void store8(float* p, const float (&x)[8])
{
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(p)), "f"(x[0]),
                 "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]) : "memory");
}

__device__ __forceinline__ void load8(const uint16_t* p, float (&x)[8])
{
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[2 * j] = u2f(w[j] << 16); x[2 * j + 1] = u2f(w[j] & 0xffff0000U); }
}

__device__ __forceinline__ void store8(uint16_t* p, const float (&x)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = abx::pack_bf16_rne(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
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
        load8(p, x);
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
    if (vec && cnt == 8) {
        store8(p, x);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) if (k < cnt) p[k] = (uint16_t)abx::pack_bf16_rne(x[k], 0.0f);
    }
}

// ---- pairs -----------------------------------------------------------------------------------------
// Two values per FP32 instruction, each rounded as the scalar instruction rounds it.

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

// A product that an addition takes, rounded by itself: the assembler contracts mul.rn.f32x2 and add.rn.f32x2 into one
// FMA (-fmad=false notwithstanding), but not an FMA whose third operand, -0, it cannot see: a kernel argument.
__device__ __forceinline__ f2x term2(f2x a, f2x b, f2x minus_zero) { return fma2(a, b, minus_zero); }

__device__ __forceinline__ f2x add2_down(f2x a, f2x b)
{
    f2x d;
    asm("add.rm.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ f2x sub2(f2x a, f2x b) { return fma2(b, both(-1.0f), a); }

__device__ __forceinline__ void pairs(const float (&x)[8], f2x (&p)[4])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = pk2(x[2 * j], x[2 * j + 1]);
}

__device__ __forceinline__ void singles(const f2x (&p)[4], float (&x)[8])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) up2(p[j], x[2 * j], x[2 * j + 1]);
}

// the first n of a pair, 0 for the others
__device__ __forceinline__ f2x first_of(f2x x, int n)
{
    float a, b;
    up2(x, a, b);
    return pk2(n > 0 ? a : 0.0f, n > 1 ? b : 0.0f);
}

// Root and quotient by Newton's iteration from the hardware's approximations, with Markstein's last step: the exact
// remainder by FMA, times the reciprocal, added to the approximation, rounds correctly (P. Markstein, IBM J. Res.
// Dev. 34(1), 1990).  In pairs that is a third of the instructions of the scalar IEEE operations, which otherwise
// take a quarter of the kernel.  The remainder has to be exact, a multiple of 2^-149, and the quotient a normal number:
// `update` uses them for a second moment that is 0 or in [2^-100, 2^48 (1 - b2)), a first one that is 0 or at least 2^-100
// and a divisor of [2^-60, 2^25], and the IEEE operations for a lane's eight values where one is outside.  (A first moment of 2^64 or
// more, which no step leaves beside such a second one, has no test of its own.)  The tests compare every float as a root's
// operand, and quotients of moments from 2^-149 on, with results in 64 bits.
__device__ __forceinline__ f2x sqrt2(f2x x)
{
    float a, b, ya, yb;
    up2(add2(x, both(0x1p-126f)), a, b);   // no change above 2^-100, and a finite reciprocal root of 0
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(ya) : "f"(a));
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(yb) : "f"(b));
    const f2x y = pk2(ya, yb), s = mul2(x, y), h = mul2(y, both(0.5f));
    float sa, sb;
    up2(x, a, b);
    up2(s, sa, sb);
    return fma2(pk2(__fmaf_rn(-sa, sa, a), __fmaf_rn(-sb, sb, b)), h, s);
}

__device__ __forceinline__ f2x quotient2(f2x x, f2x d)
{
    float a, b, ya, yb;
    up2(d, a, b);
    asm("rcp.approx.f32 %0, %1;" : "=f"(ya) : "f"(a));
    asm("rcp.approx.f32 %0, %1;" : "=f"(yb) : "f"(b));
    const f2x n = mul2(d, both(-1.0f)), y0 = pk2(ya, yb);
    const f2x y = fma2(y0, fma2(n, y0, both(1.0f)), y0);
    const f2x q = mul2(x, y);
    return fma2(fma2(n, q, x), y, q);
}

// ---- the 8-bit block format ----------------------------------------------------------------------

// Bytes become floats by way of the significand of 2^23 + byte: one byte permute and one exact subtraction each.
__device__ __forceinline__ f2x bytes2(uint32_t w, int k)
{
    return pk2(u2f(__byte_perm(w, 0x4b000000U, 0x7440 + k)), u2f(__byte_perm(w, 0x4b000000U, 0x7441 + k)));
}

__device__ __forceinline__ void decode_m(uint2 codes, float s, f2x (&m)[4])
{
    const uint32_t w[2] = {codes.x ^ 0x80808080U, codes.y ^ 0x80808080U};   // code + 128
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = mul2(add2(bytes2(w[j >> 1], 2 * (j & 1)), both(-8388736.0f)), both(s));
}

__device__ __forceinline__ void decode_v(uint2 codes, float s, f2x (&v)[4])
{
    const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f2x r = mul2(add2(bytes2(w[j >> 1], 2 * (j & 1)), both(-8388608.0f)), both(s));
        v[j] = mul2(r, r);
    }
}

// The block's largest magnitude; a NaN's bits are above every number's, so it is a NaN if any value is.
__device__ __forceinline__ float block_max(const f2x (&x)[4])
{
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a, b;
        up2(x[j], a, b);
        asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(a), "f"(b));
    }
    return u2f(__reduce_max_sync(0xffffffffU, f2u(m)));
}

constexpr float kBelow127 = 126.99999237060546875f, kBelow255 = 254.9999847412109375f;

struct BlockScales {
    float to_m, to_root;   // from values to codes
    float m, root;         // stored
};

// The numerators are the floats next below the largest codes: value * (below / top) then never rounds above that code.
// A block under 2^-100 is stored as zeros: below / top could overflow.  top not finite: the stored scale is NaN.
__device__ __forceinline__ BlockScales block_scales(float top_m, float top_root)
{
    constexpr float kLeast = 0x1p-100f, kMost = 3.402823466e38f;
    BlockScales s;
    if (top_m >= 0x1p-60f && top_m <= 0x1p90f && top_root >= 0x1p-60f && top_root <= 0x1p90f) {
        up2(quotient2(pk2(kBelow127, kBelow255), pk2(top_m, top_root)), s.to_m, s.to_root);
        s.m = __fmul_rn(top_m, 1.0f / 127.0f);
        s.root = __fmul_rn(top_root, 1.0f / 255.0f);
        return s;
    }
    s.to_m = top_m <= kLeast ? 0.0f : __fdiv_rn(kBelow127, top_m);
    s.to_root = top_root <= kLeast ? 0.0f : __fdiv_rn(kBelow255, top_root);
    s.m = top_m <= kLeast ? 0.0f : top_m <= kMost ? __fmul_rn(top_m, 1.0f / 127.0f) : u2f(0x7fffffffU);
    s.root = top_root <= kLeast ? 0.0f : top_root <= kMost ? __fmul_rn(top_root, 1.0f / 255.0f) : u2f(0x7fffffffU);
    return s;
}

constexpr float kWhole = 12582912.0f;   // 1.5 * 2^23: a sum with it has the addend, rounded, in its low bits

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// 16 random bits as a float of [0, 1): 2^23 + bits, scaled and shifted in one exact FMA.
template <int HIGH>
__device__ __forceinline__ f2x uniform2(uint32_t r0, uint32_t r1)
{
    const f2x x = pk2(u2f(__byte_perm(r0, 0x4b000000U, HIGH ? 0x7432 : 0x7410)),
                      u2f(__byte_perm(r1, 0x4b000000U, HIGH ? 0x7432 : 0x7410)));
    return fma2(x, both(0x1p-16f), both(-128.0f));
}

template <bool SR>
__device__ __forceinline__ uint2 encode_m(const f2x (&m)[4], float f, const uint32_t (&r)[8], f2x minus_zero)
{
    float q[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f2x x = term2(m[j], both(f), minus_zero);
        const f2x z = SR ? add2_down(add2(x, uniform2<0>(r[2 * j], r[2 * j + 1])), both(kWhole))   // floor(x + u)
                         : add2(x, both(kWhole));
        up2(z, q[2 * j], q[2 * j + 1]);
    }
    return make_uint2(pack4(f2u(q[0]), f2u(q[1]), f2u(q[2]), f2u(q[3])), pack4(f2u(q[4]), f2u(q[5]), f2u(q[6]), f2u(q[7])));
}

// Codes of which those that are 0 become 1, but for the bytes that are 1 in `zeros`: code 0 is for 0 alone.
__device__ __forceinline__ uint32_t at_least_one(uint32_t codes, uint32_t zeros)
{
    // the sign bits of 0 bytes; a borrow also marks a byte of 1 above one, which keeps its value
    const uint32_t none = (codes - 0x01010101U) & ~codes & 0x80808080U;
    return codes | (none >> 7 & ~zeros);
}

template <bool SR>
__device__ __forceinline__ uint2 encode_v(const f2x (&root)[4], float f, const uint32_t (&r)[8], const uint32_t (&zeros)[2],
                                          f2x minus_zero)
{
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float za, zb;
        const f2x x = term2(root[j], both(f), minus_zero);
        if (SR) {
            const f2x z = add2_down(x, both(kWhole)), q = add2(z, both(-kWhole));
            const f2x part = mul2(sub2(x, q), add2(x, q));
            const f2x step = mul2(uniform2<1>(r[2 * j], r[2 * j + 1]), fma2(q, both(2.0f), both(1.0f)));
            float da, db;
            up2(z, za, zb);
            up2(sub2(step, part), da, db);   // negative: up
            c[2 * j] = f2u(za) + (f2u(da) >> 31);
            c[2 * j + 1] = f2u(zb) + (f2u(db) >> 31);
        } else {
            up2(add2(x, both(kWhole)), za, zb);
            c[2 * j] = f2u(za);
            c[2 * j + 1] = f2u(zb);
        }
    }
    return make_uint2(at_least_one(pack4(c[0], c[1], c[2], c[3]), zeros[0]),
                      at_least_one(pack4(c[4], c[5], c[6], c[7]), zeros[1]));
}

// ---- the step ------------------------------------------------------------------------------------

template <int N>
__device__ __forceinline__ int find_item(const Args<N>& a, int lo, int tile)
{
    int hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].tile_begin <= tile) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Where a lane's eight values lie.  A CTA's tiles of a tensor are a fixed distance apart, so the addresses are worked
// out once per tensor and moved on from tile to tile.
template <bool I8, typename W>
struct Lane {
    W* w;
    const W* g;
    float* master;
    uint8_t* m;
    uint8_t* v;
    float* m_scale;
    float* v_scale;
    uint32_t place;   // of the first value in its tensor (low 32 bits), which the rounding's random words go by

    __device__ __forceinline__ Lane(const Item& t, int64_t at)
    {
        constexpr int kMoment = I8 ? 1 : 4;   // bytes
        at += threadIdx.x * 8;
        w = static_cast<W*>(t.w) + at;
        g = static_cast<const W*>(t.g) + at;
        master = t.master + at;
        m = static_cast<uint8_t*>(t.m) + at * kMoment;
        v = static_cast<uint8_t*>(t.v) + at * kMoment;
        m_scale = t.m_scale + at / kBlock;
        v_scale = t.v_scale + at / kBlock;
        place = (uint32_t)at;
    }
    __device__ __forceinline__ void advance(int64_t by)
    {
        constexpr int kMoment = I8 ? 1 : 4;
        w += by;
        if constexpr (!I8) g += by;
        if constexpr (sizeof(W) == 2) master += by;
        m += by * kMoment;
        v += by * kMoment;
        if constexpr (I8) {
            m_scale += by / kBlock;
            v_scale += by / kBlock;
        }
        place += (uint32_t)by;
    }
};

struct Constants {
    float scale, b1, omb1, b2, omb2, eps;
    f2x minus_zero;
    uint32_t plain_low, plain_high, zero_is_plain;
};

// Eight values of a lane as they are stored.
template <bool I8, typename W> struct Loaded;
template <typename W> struct Loaded<false, W> { float g[8], p[8], m[8], v[8]; };
template <typename W> struct Loaded<true, W> { float g[8], p[8]; uint2 m, v; float sm, sv; };

// cnt of the lane's values are valid (8 where FULL).
template <bool I8, bool FULL, typename W>
__device__ __forceinline__ void load(Loaded<I8, W>& x, const Lane<I8, W>& t, int cnt, bool vec)
{
    constexpr bool kMaster = sizeof(W) == 2;
    if constexpr (FULL) load8(t.g, x.g);
    else load8(t.g, cnt, vec, x.g);
    if constexpr (kMaster) load8(t.master, x.p);
    else if constexpr (FULL) load8(t.w, x.p);
    else load8(t.w, cnt, vec, x.p);
    if constexpr (I8) {
        x.m = *reinterpret_cast<const uint2*>(t.m);
        x.v = *reinterpret_cast<const uint2*>(t.v);
        x.sm = *t.m_scale;
        x.sv = *t.v_scale;
    } else {
        load8(reinterpret_cast<const float*>(t.m), x.m);
        load8(reinterpret_cast<const float*>(t.v), x.v);
    }
}

__device__ __forceinline__ float least_abs(float a, float b, float c)
{
    float d;
    asm("min.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

constexpr float kLeastPlain = 0x1p-100f;   // of a first moment that is not 0, and of a second one

// One block of 256 values, 8 per lane.
template <bool I8, bool SR, bool FULL, typename W>
__device__ __forceinline__ void update(const Loaded<I8, W>& in, const Lane<I8, W>& t, const Constants& k, const StepCoef& c,
                                       int cnt, bool vec)
{
    constexpr bool kMaster = sizeof(W) == 2;
    const f2x nz = k.minus_zero;
    float x[8];
    f2x g[4], p[4], m[4], v[4], root[4], q[4];
    pairs(in.g, g);
    pairs(in.p, p);
    if constexpr (I8) {
        decode_m(in.m, in.sm, m);
        decode_v(in.v, in.sv, v);
    } else {
        pairs(in.m, m);
        pairs(in.v, v);
    }
    uint32_t low = 0xffffffffU, high = 0;   // the extremes of v's bits
    float least = 1.0f;                     // ... and of |m|
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f2x gj = mul2(g[j], both(k.scale));
        m[j] = add2(term2(m[j], both(k.b1), nz), term2(gj, both(k.omb1), nz));
        v[j] = add2(term2(v[j], both(k.b2), nz), term2(mul2(gj, both(k.omb2)), gj, nz));
        float v0, v1;
        up2(v[j], v0, v1);
        low = __vimin3_u32(low, f2u(v0), f2u(v1));
        high = __vimax3_u32(high, f2u(v0), f2u(v1));
        float m0, m1;
        up2(m[j], m0, m1);
        least = least_abs(least, m0, m1);
        root[j] = sqrt2(v[j]);
        q[j] = quotient2(m[j], add2(term2(root[j], both(c.inv_sqrt_bc2), nz), both(k.eps)));
    }
    uint32_t zeros[2] = {0, 0};   // a 1 in the byte of each v that is 0
    if (__builtin_expect(low < k.plain_low || high >= k.plain_high || least < kLeastPlain, 0)) {
        bool ieee = !k.zero_is_plain || high >= k.plain_high;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v0, v1, m0, m1;
            up2(v[j], v0, v1);
            up2(m[j], m0, m1);
            zeros[j >> 1] |= ((f2u(v0) == 0 ? 1U : 0U) | (f2u(v1) == 0 ? 0x100U : 0U)) << (16 * (j & 1));
            ieee |= (f2u(v0) != 0 && f2u(v0) < k.plain_low) || (f2u(v1) != 0 && f2u(v1) < k.plain_low)
                    || (m0 != 0.0f && fabsf(m0) < kLeastPlain) || (m1 != 0.0f && fabsf(m1) < kLeastPlain);
        }
        if (ieee) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v0, v1, m0, m1;
                up2(v[j], v0, v1);
                up2(m[j], m0, m1);
                v0 = __fsqrt_rn(v0);
                v1 = __fsqrt_rn(v1);
                root[j] = pk2(v0, v1);
                q[j] = pk2(__fdiv_rn(m0, __fadd_rn(__fmul_rn(v0, c.inv_sqrt_bc2), k.eps)),
                           __fdiv_rn(m1, __fadd_rn(__fmul_rn(v1, c.inv_sqrt_bc2), k.eps)));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = sub2(term2(p[j], both(c.decay), nz), term2(q[j], both(c.step_size), nz));
    if constexpr (!FULL) {   // beyond the tensor's end the state stays zero
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[j] = first_of(p[j], cnt - 2 * j);
            m[j] = first_of(m[j], cnt - 2 * j);
            if constexpr (I8) root[j] = first_of(root[j], cnt - 2 * j);
            else v[j] = first_of(v[j], cnt - 2 * j);   // not 0 there by itself: 0 times a scale that is not finite
        }
        if (cnt < 4) zeros[0] |= 0x01010101U << (8 * cnt);
        zeros[1] |= cnt <= 4 ? 0x01010101U : cnt < 8 ? 0x01010101U << (8 * (cnt - 4)) : 0U;
    }
    singles(p, x);
    if constexpr (kMaster) store8(t.master, x);
    if constexpr (FULL) store8(t.w, x);
    else store8(t.w, cnt, vec, x);
    if constexpr (I8) {
        uint32_t r[8];
        if constexpr (SR) {
            uint32_t r0[4], r1[4];
            abx::hash4(t.place, c.stream, r0);
            abx::hash4(t.place + 4, c.stream, r1);
#pragma unroll
            for (int i = 0; i < 4; ++i) { r[i] = r0[i]; r[4 + i] = r1[i]; }
        }
        const BlockScales s = block_scales(block_max(m), block_max(root));
        *reinterpret_cast<uint2*>(t.m) = encode_m<SR>(m, s.to_m, r, nz);
        *reinterpret_cast<uint2*>(t.v) = encode_v<SR>(root, s.to_root, r, zeros, nz);
        if (threadIdx.x % 32 == 0) {
            *t.m_scale = s.m;
            *t.v_scale = s.root;
        }
    } else {
        singles(m, x);
        store8(reinterpret_cast<float*>(t.m), x);
        singles(v, x);
        store8(reinterpret_cast<float*>(t.v), x);
    }
}

// 8-bit moments: a warp's blocks travel through shared memory, kStages - 1 of them under way while one is computed.
// That needs no registers for what is under way, and the copies of a warp are contiguous.
template <typename W>
struct Ring {
    static constexpr int kStages = 3;
    static constexpr int kP = 0, kG = kP + 4 * kBlock, kM = kG + (int)sizeof(W) * kBlock, kV = kM + kBlock, kS = kV + kBlock;
    static constexpr int kBytes = kS + 16;
};

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from)
{
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(__cvta_generic_to_global(from)) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(__cvta_generic_to_global(from)), "n"(BYTES)
                     : "memory");
}

// What a lane copies of its warp's blocks: neighbouring lanes copy neighbouring pieces.
template <typename W>
struct Fetch {
    static constexpr int kPer = 16 / (int)sizeof(W);
    const float* p;
    const W* g;
    const uint8_t* m;
    const uint8_t* v;
    const float* m_scale;
    const float* v_scale;

    __device__ __forceinline__ Fetch(const Item& t, int64_t at)
    {
        const uint32_t lane = threadIdx.x % 32;
        at += threadIdx.x / 32 * kBlock;
        if constexpr (sizeof(W) == 2) p = t.master;
        else p = static_cast<const float*>(t.w);
        p += at + lane * 4;
        g = static_cast<const W*>(t.g) + at + lane * kPer;
        m = static_cast<const uint8_t*>(t.m) + at + lane * 8;
        v = static_cast<const uint8_t*>(t.v) + at + lane * 8;
        m_scale = t.m_scale + at / kBlock;
        v_scale = t.v_scale + at / kBlock;
    }
    // Start the copies of this block, and move on to the next.
    __device__ __forceinline__ void start(uint32_t to, int64_t by)
    {
        using R = Ring<W>;
        const uint32_t lane = threadIdx.x % 32;
        copy_async<16>(to + R::kP + lane * 16, p);
        copy_async<16>(to + R::kP + 512 + lane * 16, p + 128);
        copy_async<16>(to + R::kG + lane * 16, g);
        if constexpr (sizeof(W) == 4) copy_async<16>(to + R::kG + 512 + lane * 16, g + 128);
        copy_async<8>(to + R::kM + lane * 8, m);
        copy_async<8>(to + R::kV + lane * 8, v);
        if (lane == 0) {
            copy_async<4>(to + R::kS, m_scale);
            copy_async<4>(to + R::kS + 4, v_scale);
        }
        p += by;
        g += by;
        m += by;
        v += by;
        m_scale += by / kBlock;
        v_scale += by / kBlock;
    }
};

__device__ __forceinline__ void shared8(const uint8_t* p, float (&x)[8])
{
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

template <typename W>
__device__ __forceinline__ void take(Loaded<true, W>& x, const uint8_t* from)
{
    using R = Ring<W>;
    const uint32_t lane = threadIdx.x % 32;
    shared8(from + R::kP + lane * 32, x.p);
    if constexpr (sizeof(W) == 4) shared8(from + R::kG + lane * 32, x.g);
    else load8(reinterpret_cast<const uint16_t*>(from + R::kG + lane * 16), x.g);
    x.m = *reinterpret_cast<const uint2*>(from + R::kM + lane * 8);
    x.v = *reinterpret_cast<const uint2*>(from + R::kV + lane * 8);
    x.sm = *reinterpret_cast<const float*>(from + R::kS);
    x.sv = *reinterpret_cast<const float*>(from + R::kS + 4);
}

// W: the weights' and gradients' type (float, or uint16_t for bf16 bits with an fp32 master).  A warp takes a block of
// each of its CTA's tiles.
template <bool I8, bool SR, typename W, int N>
__global__ void __launch_bounds__(kThreads, kStepCtas<I8>) step_kernel(const __grid_constant__ Args<N> a)
{
    using R = Ring<W>;
    __shared__ __align__(16) uint8_t ring[I8 ? kWarps * R::kStages * R::kBytes : 16];
    __shared__ bool last;
    // skip is a flag as loss scalers write it; a norm that is not finite says the same of the gradients
    if (a.skip != nullptr && !(*a.skip == 0.0f)) return;
    if (a.norm != nullptr && !(fabsf(*a.norm) <= 3.402823466e38f)) return;
    const Constants constants{a.g_scale != nullptr ? *a.g_scale : 1.0f, a.b1, a.omb1, a.b2, a.omb2, a.eps, both(a.minus_zero),
                              a.plain_low, a.plain_high, a.zero_is_plain};
    const uint32_t mine = threadIdx.x / 32 * kBlock;   // the warp's block in a tile
    uint8_t* const slots = ring + threadIdx.x / 32 * (R::kStages * R::kBytes);
    const int64_t apart = (int64_t)gridDim.x * kTile;
    int item = 0;
    for (int tile = blockIdx.x; tile < a.tiles;) {   // from tensor to tensor
        item = find_item(a, item, tile);
        const Item& t = a.t[item];
        const int end = item + 1 < a.count ? a.t[item + 1].tile_begin : a.tiles;
        const StepCoef c = step_coef(a, t);
        const bool vec = t.index_vec & 1;
        int64_t at = (int64_t)(tile - t.tile_begin) * kTile;
        Lane<I8, W> here(t, at);
        // this CTA's whole tiles that allow vector access
        const int64_t room = vec ? t.n - kTile - at : -1;
        const int whole = room < 0 ? 0 : (int)(room / apart) + 1;
        if constexpr (I8) {
            if (whole > 0) {
                Fetch<W> ahead(t, at);
                const auto fetch = [&](int k) {
                    if (k < whole) ahead.start((uint32_t)__cvta_generic_to_shared(slots + k % R::kStages * R::kBytes), apart);
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
#pragma unroll
                for (int k = 0; k < R::kStages - 1; ++k) fetch(k);
                for (int k = 0; k < whole; ++k) {
                    fetch(k + R::kStages - 1);
                    asm volatile("cp.async.wait_group %0;" ::"n"(R::kStages - 1) : "memory");
                    __syncwarp();   // the other lanes' copies too
                    Loaded<I8, W> x;
                    take(x, slots + k % R::kStages * R::kBytes);
                    update<I8, SR, true, W>(x, here, constants, c, 8, true);
                    here.advance(apart);
                    __syncwarp();   // every lane has read this slot
                }
            }
        } else {
            for (int k = 0; k < whole; ++k) {
                Loaded<I8, W> x;
                load<I8, true, W>(x, here, 8, true);
                update<I8, SR, true, W>(x, here, constants, c, 8, true);
                here.advance(apart);
            }
        }
        tile += whole * gridDim.x;
        at += whole * apart;
        for (; tile < end; tile += gridDim.x, at += apart) {
            if (at + mine >= t.n) continue;
            const Lane<I8, W> last_lane(t, at);
            const int64_t rest = t.n - at - (int64_t)threadIdx.x * 8;
            const int cnt = rest < 0 ? 0 : rest > 8 ? 8 : (int)rest;
            Loaded<I8, W> x;
            load<I8, false, W>(x, last_lane, cnt, vec);
            update<I8, SR, false, W>(x, last_lane, constants, c, cnt, vec);
        }
    }
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
    float minus_zero;
};

// A warp takes four blocks at a time, so that enough loads are under way.
template <bool V>
__global__ void __launch_bounds__(kThreads) i8_decode(const I8Args a)
{
    constexpr int kAtOnce = 4;
    const int lane = threadIdx.x & 31;
    const bool vec = (reinterpret_cast<uintptr_t>(a.values) & 31) == 0;
    const int64_t stride = (int64_t)gridDim.x * kWarps * kAtOnce;
    for (int64_t b = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * kAtOnce; b < a.blocks; b += stride) {
        uint2 c[kAtOnce];
        float s[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (b + j < a.blocks) {
                c[j] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.codes) + (b + j) * kBlock + lane * 8);
                s[j] = a.scales[b + j];
            }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const int64_t i0 = (b + j) * kBlock + lane * 8, left = a.n - i0;
            if (b + j >= a.blocks || left <= 0) break;
            float x[8];
            f2x y[4];
            if constexpr (V) decode_v(c[j], s[j], y);
            else decode_m(c[j], s[j], y);
            singles(y, x);
            store8(a.values + i0, left < 8 ? (int)left : 8, vec, x);
        }
    }
}

// Nearest codes.  A negative second moment counts as 0.
template <bool V>
__global__ void __launch_bounds__(kThreads) i8_encode(const I8Args a)
{
    const int lane = threadIdx.x & 31;
    const bool vec = (reinterpret_cast<uintptr_t>(a.values) & 31) == 0;
    for (int64_t b = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); b < a.blocks; b += (int64_t)gridDim.x * kWarps) {
        const int64_t i0 = b * kBlock + lane * 8, left = a.n - i0;
        float x[8];
        load8(a.values + i0, left >= 8 ? 8 : (left > 0 ? (int)left : 0), vec, x);
        if constexpr (V) {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = __fsqrt_rn(x[k] < 0.0f ? 0.0f : x[k]);
        }
        const uint32_t none[8] = {};
        f2x y[4];
        pairs(x, y);
        const float top = block_max(y);
        const BlockScales s = block_scales(top, top);
        uint2 c;
        if constexpr (V) {
            uint32_t zeros[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 8; ++k) zeros[k >> 2] |= (x[k] > 0.0f ? 0U : 1U) << (8 * (k & 3));
            c = encode_v<false>(y, s.to_root, none, zeros, both(a.minus_zero));
        }
        else c = encode_m<false>(y, s.to_m, none, both(a.minus_zero));
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.codes) + i0) = c;
        if (lane == 0) a.scales[b] = V ? s.root : s.m;
    }
}

// ---- host side ---------------------------------------------------------------------------------------

bool off(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }

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
    if (off(t.m, 32) || off(t.v, 32) || (t.dtype == ABX_DT_BF16 && off(t.master, 32))) return ABX_E_ALIGN;
    if (h.moments == ABX_DT_I8 && (off(t.m_scale, 4) || off(t.v_scale, 4))) return ABX_E_ALIGN;
    return ABX_OK;
}

// CTAs of a kernel that are resident on the current device, asked for once per device.
template <auto KERNEL>
int resident_ctas(int* out)
{
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];
    int dev = 0, sms = 0, per = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const bool keep = e == cudaSuccess && dev < kDevices;
    if (keep && (*out = known[dev].load(std::memory_order_relaxed)) > 0) return ABX_OK;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, (const void*)KERNEL, kThreads, 0);
    if (e != cudaSuccess) return abx::set_error("launch geometry", e);
    *out = sms * (per > 0 ? per : 1);
    if (keep) known[dev].store(*out, std::memory_order_relaxed);
    return ABX_OK;
}

template <bool I8, bool SR, typename W, int N>
int launch_step(const Args<N>& a, int32_t max_ctas, cudaStream_t st)
{
    int grid = 0;
    if (int rc = resident_ctas<step_kernel<I8, SR, W, N>>(&grid)) return rc;
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
int run_batch(const abx_graph_tensor* t, const int32_t* order, int32_t count, const abx_graph_step& h,
              uint32_t* ticket, int32_t max_ctas, cudaStream_t st)
{
    static thread_local Args<N> a;   // kept off the stack
    a.lr = h.lr; a.b1d = h.beta1; a.b2d = h.beta2; a.weight_decay = h.weight_decay;
    a.lr_ptr = h.lr_ptr; a.lr_f64 = h.lr_f64;
    a.g_scale = h.g_scale; a.skip = h.skip; a.norm = h.norm; a.ticket = ticket;
    a.count = count; a.seed = h.seed;
    a.b1 = (float)h.beta1; a.omb1 = (float)(1.0 - h.beta1);
    a.b2 = (float)h.beta2; a.omb2 = (float)(1.0 - h.beta2);
    a.eps = (float)h.eps;
    a.minus_zero = -0.0f;
    // The divisor is sqrt(v) c + eps, c at most 1 / sqrt(1 - b2): below 2^24 + 2^24 where v is below 2^48 (1 - b2).
    const float high = (float)((1.0 - h.beta2) * 0x1p48), low = kLeastPlain;
    std::memcpy(&a.plain_low, &low, 4);
    std::memcpy(&a.plain_high, &high, 4);
    if (!(a.eps >= 0.0f && a.eps <= 0x1p24f)) a.plain_high = 0;
    a.zero_is_plain = a.eps >= 0x1p-60f;
    int64_t next = 0;
    for (int32_t j = 0; j < count; ++j) {
        const abx_graph_tensor& s = t[order[j]];
        const uintptr_t wide = s.dtype == ABX_DT_F32 ? 32 : 16;   // bytes of 8 values
        const uint32_t vec = !off(s.w, wide) && !off(s.g, wide);
        a.t[j] = Item{s.w, s.g, s.master, s.m, s.v, s.m_scale, s.v_scale, s.step, s.n, (int32_t)next, s.index << 1 | vec};
        next += tiles_of(s.n);
    }
    a.tiles = (int32_t)next;
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
int i8_run(void* stream, void* codes, float* scales, float* values, int64_t n, int32_t role, int at_once, const char* what)
{
    if (int rc = i8_check(codes, scales, values, n, role)) return rc;
    if (n == 0) return ABX_OK;
    const I8Args a{codes, scales, values, n, (n + kBlock - 1) / kBlock, -0.0f};
    int grid = 0;
    if (int rc = role ? resident_ctas<KV>(&grid) : resident_ctas<KM>(&grid)) return rc;
    const int64_t need = (a.blocks + kWarps * at_once - 1) / (kWarps * at_once);
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
                const int64_t more = tiles_of(tensors[i].n);
                if (tiles + more > kMaxTiles) break;
                order[count++] = i;
                tiles += more;
            }
            if (count == 0) break;   // only other dtypes and empty tensors were left
            const int rc = count <= kFew ? run_batch<kFew>(tensors, order, count, h, ticket, max_ctas, st)
                                         : run_batch<kMany>(tensors, order, count, h, ticket, max_ctas, st);
            if (rc) return rc;
        }
    }
    return ABX_OK;
}

ABX_API int abx_i8_decode(void* stream, const void* codes, const float* scales, float* values, int64_t n, int32_t role)
{
    return i8_run<i8_decode<false>, i8_decode<true>>(stream, const_cast<void*>(codes), const_cast<float*>(scales), values,
                                                     n, role, 4, "i8_decode launch");
}

ABX_API int abx_i8_encode(void* stream, const float* values, void* codes, float* scales, int64_t n, int32_t role)
{
    return i8_run<i8_encode<false>, i8_encode<true>>(stream, codes, scales, const_cast<float*>(values), n, role, 1,
                                                     "i8_encode launch");
}
