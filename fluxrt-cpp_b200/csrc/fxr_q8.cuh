// fxr_q8.cuh — the 8-bit spatial cache (sm_100a): codes, scales and the kernels that move rows.
//
// A head vector x (128 values of one token's K' or V) is held as 128 codes of 8 bits and one scale of
// the frame's 16-bit type T:
//   s    = up_T(max|x| / Q)            Q = 127 (int8) or 448 (e4m3); up_T rounds up to T
//   code = rint(x / s) in [-127, 127]  or  e4m3(x / s), nearest even, saturating
//   read = T(code * s)                 one rounding
// The scale is a number of T, so that the read-back is one packed multiply with one rounding, in the
// read kernel and in the attention alike; rounding it up keeps |x / s| <= Q, at a cost of at most
// 2^-8 (bf16) or 2^-11 (f16) of the range. Where Q * s would pass the largest f16 the scale is
// rounded down instead and the largest codes saturate. A vector of zeros has scale 0; one that holds
// an infinity or NaN has scale NaN and codes 0, and reads back as NaN.
//   q8_write_kernel     executed rows: gather + QK-RMSNorm + RoPE + quantised cache rows, or (raw)
//                       the quantised rows of an attention-ready 16-bit cache
//   q8_read_kernel      rows back in 16 bits
//   q8_expand_kernel    whole caches in 16 bits, for the attention over many rows
//   q8_restore_kernel   puts back the cache rows of mask==1 tokens
#pragma once

#include <cuda_fp8.h>

#include "fxr_mem_kernels.cuh"

namespace fxr {
namespace q8 {

constexpr int kInt8 = 0, kE4m3 = 1;

// One cache, as a kernel argument. Code rows: [n_rows, ld] bytes; scales: [n_heads, ld_scale] of T.
struct Cache {
    uint8_t* k;
    uint8_t* v;
    void* ks;
    void* vs;
    int64_t ld, ld_scale;
};

// ---- codes --------------------------------------------------------------------------------------
template <int F> __device__ __forceinline__ constexpr float top_code() { return F == kInt8 ? 127.f : 448.f; }

template <typename T> __device__ __forceinline__ float scale_up(float t);
template <> __device__ __forceinline__ float scale_up<__nv_bfloat16>(float t) {
    return __uint_as_float((__float_as_uint(t) + 0xffffu) & 0xffff0000u);   // t >= 0
}
template <> __device__ __forceinline__ float scale_up<__half>(float t) { return __half2float(__float2half_ru(t)); }

// (largest T) / 128 or / 448, rounded down to T.
template <typename T, int F> __device__ __forceinline__ constexpr float scale_cap() {
    constexpr bool bf16 = StoreT<T>::kUmmaFormat == 1;
    return F == kInt8 ? (bf16 ? 0x1.fep+120f : 511.75f) : (bf16 ? 0x1.22p+119f : 146.125f);
}

// Whether s is a scale that the write stores for a finite vector (every code times it is finite).
template <typename T, int F> __device__ __forceinline__ bool valid_scale(float s) { return fabsf(s) <= scale_cap<T, F>(); }

// Scale of a head vector whose largest magnitude is amax (infinite or NaN where an element is).
template <typename T, int F>
__device__ __forceinline__ float scale_of(float amax) {
    if (!(amax < INFINITY)) return __uint_as_float(0x7fc00000u);
    return fminf(scale_up<T>(__fdiv_rn(amax, top_code<F>())), scale_cap<T, F>());
}

// Maximum that is NaN where an operand is.
__device__ __forceinline__ float max3n(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max2n(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 f2add(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}

// Codes of 4 values as 4 bytes. x / s is taken as x times the rounded 1 / s, off by at most 2^-22
// relative (1.5e-5 of a code). kExact (x of T): such a quotient of two numbers of T that is not half way
// between two codes is farther from there than 2.4e-4 of a code (int8; the numerator of the difference
// is a whole multiple of the smaller unit) or 2^-16 relative (e4m3), so rounding it first to a multiple
// of 2^-13, or to 18 bits, puts the half-way cases, and only those, exactly half way, and the
// nearest-even rounding that follows is that of the true quotient. (Divisions took half of the write
// kernel's instructions.)
template <int F, bool kExact>
__device__ __forceinline__ uint32_t encode4(float2 a, float2 b, float r, bool clamp) {
    float2 y[2] = {f2mul(a, make_float2(r, r)), f2mul(b, make_float2(r, r))};
    if (F == kInt8) {
        // in 1.5 * 2^23 + y the low byte of the bits is y's whole number, two's complement
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (clamp) y[e] = make_float2(fminf(fmaxf(y[e].x, -127.f), 127.f), fminf(fmaxf(y[e].y, -127.f), 127.f));
            if (kExact) y[e] = f2add(f2add(y[e], make_float2(1536.f, 1536.f)), make_float2(-1536.f, -1536.f));
            y[e] = f2add(y[e], make_float2(12582912.f, 12582912.f));
        }
        return __byte_perm(__byte_perm(__float_as_uint(y[0].x), __float_as_uint(y[0].y), 0x0040),
                           __byte_perm(__float_as_uint(y[1].x), __float_as_uint(y[1].y), 0x0040), 0x5410);
    } else {
        if (kExact) {      // c - (c - y) with c = (2^6 + 1) y is y in 18 bits
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 c = f2mul(y[e], make_float2(65.f, 65.f));
                y[e] = f2add(c, f2mul(f2add(c, make_float2(-y[e].x, -y[e].y)), make_float2(-1.f, -1.f)));
            }
        }
        return (uint32_t)__nv_cvt_float2_to_fp8x2(y[0], __NV_SATFINITE, __NV_E4M3) |
               ((uint32_t)__nv_cvt_float2_to_fp8x2(y[1], __NV_SATFINITE, __NV_E4M3) << 16);
    }
}

__device__ __forceinline__ __nv_bfloat162 as_bf(uint32_t u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); }
__device__ __forceinline__ __half2 as_h(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ uint32_t bits(const __nv_bfloat162& x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ uint32_t bits(const __half2& x) { return *reinterpret_cast<const uint32_t*>(&x); }
template <typename T> __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t mul2<__nv_bfloat16>(uint32_t a, uint32_t b) { return bits(__hmul2(as_bf(a), as_bf(b))); }
template <> __device__ __forceinline__ uint32_t mul2<__half>(uint32_t a, uint32_t b) { return bits(__hmul2(as_h(a), as_h(b))); }

// Codes -> T(code * s), pairs of T at a time. What bounds a decoder is the integer pipe, which runs at
// half the rate of the FMA pipe (the attention's converters share both with the softmax warps), so as
// much as can be is left to packed 16-bit arithmetic:
//   int8 -> bf16: a permute puts byte x ^ 0x80 under the constant 0x42, the bf16 number a = 64 + x / 2
//     for x >= 0 and 64 + x / 4 for x < 0. Then t = 2 s a - 128 s (one fma, one rounding) is s x for
//     x >= 0 and s x / 2 otherwise, and t - max(0, -t) is s x for both: rounding commutes with the
//     factor 2, so the result is the one rounding of s x.
//   int8 -> f16:  0x6400 | (x ^ 0x80) is 1024 + 128 + x, exactly: subtract, multiply.
//   e4m3 -> f16:  sign, exponent and mantissa fields moved into place give the value times 2^-8 (also
//     where it is subnormal); the scale's multiplier holds the 2^8. The permute doubles the byte, so
//     that the sign is in place already and the rest a left shift away, which the FMA pipe does.
//   e4m3 -> bf16: the same gives the value times 2^-120; products of bf16 keep subnormal operands, so
//     a multiplication by 2^120 restores it. Where s < 2^7, as for every vector of magnitude below
//     57344, the scale's multiplier holds the 2^120 (SmallScaleDecoder).
// The codes 0x7f and 0xff, NaN in other uses of e4m3, which the write never produces, are +-480: a cache
// may hold rows that nobody wrote, and a code that decodes to NaN would reach the rows that do not see it
// (0 * NaN).
template <typename T, int F> struct Decoder;

// word(): prepares four codes, once; pair(): two of them as values.
template <> struct Decoder<__nv_bfloat16, kInt8> {
    __nv_bfloat162 two, up, mtwo, down;      // 2 s, -128 s, -2 s, 128 s
    __device__ __forceinline__ void scale(uint32_t s2) {
        const __nv_bfloat162 s = as_bf(s2);
        two = __hmul2(s, as_bf(0x40004000u));
        mtwo = __hmul2(s, as_bf(0xc000c000u));
        down = __hmul2(s, as_bf(0x43004300u));
        up = __hmul2(s, as_bf(0xc300c300u));
    }
    static __device__ __forceinline__ uint32_t word(uint32_t w) { return w ^ 0x80808080u; }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int a, int b) const {
        const uint32_t u = __byte_perm(w, 0x42424242u, (uint32_t)(a | 0x40 | (b << 8) | 0x4000));
        const __nv_bfloat162 t = __hfma2(as_bf(u), two, up), n = __hfma2_relu(as_bf(u), mtwo, down);
        return bits(__hsub2(t, n));
    }
};
template <> struct Decoder<__half, kInt8> {
    __half2 s;
    __device__ __forceinline__ void scale(uint32_t s2) { s = as_h(s2); }
    static __device__ __forceinline__ uint32_t word(uint32_t w) { return w ^ 0x80808080u; }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int a, int b) const {
        const uint32_t u = __byte_perm(w, 0x64646464u, (uint32_t)(a | 0x40 | (b << 8) | 0x4000));
        return bits(__hmul2(__hsub2(as_h(u), as_h(0x64806480u)), s));
    }
};
template <> struct Decoder<__half, kE4m3> {
    __half2 s;
    __device__ __forceinline__ void scale(uint32_t s2) { s = __hmul2(as_h(s2), as_h(0x5c005c00u)); }   // * 2^8: s <= 146.125
    static __device__ __forceinline__ uint32_t word(uint32_t w) { return w; }
    static __device__ __forceinline__ uint32_t fields(uint32_t w, int a, int b) {
        const uint32_t u = __byte_perm(w, 0u, (uint32_t)(a | (a << 4) | (b << 8) | (b << 12)));
        return ((u << 7) & 0x3f803f80u) | (u & 0x80008000u);
    }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int a, int b) const {
        return bits(__hmul2(as_h(fields(w, a, b)), s));
    }
};
template <> struct Decoder<__nv_bfloat16, kE4m3> {
    __nv_bfloat162 s;
    __device__ __forceinline__ void scale(uint32_t s2) { s = as_bf(s2); }
    static __device__ __forceinline__ uint32_t word(uint32_t w) { return w; }
    static __device__ __forceinline__ uint32_t fields(uint32_t w, int a, int b) {
        const uint32_t u = __byte_perm(w, 0u, (uint32_t)(a | (a << 4) | (b << 8) | (b << 12)));
        return ((u << 4) & 0x07f007f0u) | (u & 0x80008000u);
    }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int a, int b) const {
        return bits(__hmul2(__hmul2(as_bf(fields(w, a, b)), as_bf(0x7b807b80u)), s));
    }
};
// e4m3 -> bf16 for scales of magnitude below `limit` (or NaN): one multiplication.
struct SmallScaleDecoder {
    static constexpr float limit = 128.f;
    __nv_bfloat162 s;
    __device__ __forceinline__ void scale(uint32_t s2) { s = __hmul2(as_bf(s2), as_bf(0x7b807b80u)); }
    static __device__ __forceinline__ uint32_t word(uint32_t w) { return w; }
    __device__ __forceinline__ uint32_t pair(uint32_t w, int a, int b) const {
        return bits(__hmul2(as_bf(Decoder<__nv_bfloat16, kE4m3>::fields(w, a, b)), s));
    }
};
// The largest valid scales times 480 pass the largest T. In the attention such a product stops there (a NaN
// stays one), since an infinite V row would turn a weight of 0 into NaN.
template <typename T> __device__ __forceinline__ uint32_t to_finite2(uint32_t x);
template <> __device__ __forceinline__ uint32_t to_finite2<__nv_bfloat16>(uint32_t x) {
    return bits(__hmin2_nan(__hmax2_nan(as_bf(x), as_bf(0xff7fff7fu)), as_bf(0x7f7f7f7fu)));
}
template <> __device__ __forceinline__ uint32_t to_finite2<__half>(uint32_t x) {
    return bits(__hmin2_nan(__hmax2_nan(as_h(x), as_h(0xfbfffbffu)), as_h(0x7bff7bffu)));
}
template <typename T> struct FiniteDecoder : Decoder<T, kE4m3> {
    __device__ __forceinline__ uint32_t pair(uint32_t w, int a, int b) const {
        return to_finite2<T>(Decoder<T, kE4m3>::pair(w, a, b));
    }
};
// Decoders of the attention: `any` for every valid scale, and `small` for a tile whose scales are all of
// magnitude below `limit` (or NaN).
template <typename T, int F> struct TileDecoder {
    static constexpr bool has_limit = false;
    using any = Decoder<T, F>;
};
template <> struct TileDecoder<__nv_bfloat16, kE4m3> {
    static constexpr bool has_limit = true;
    static constexpr float limit = SmallScaleDecoder::limit;
    using any = FiniteDecoder<__nv_bfloat16>;
    using small = SmallScaleDecoder;
};
template <> struct TileDecoder<__half, kE4m3> {
    static constexpr bool has_limit = true;
    static constexpr float limit = 136.f;       // 480 * 136 = 65280
    using any = FiniteDecoder<__half>;
    using small = Decoder<__half, kE4m3>;
};

// Codes alone as a pair of f16, which holds every code exactly. word: four codes prepared by code_word;
// upper: its codes 2 and 3, not 0 and 1. e4m3 has an instruction for it, which makes 0x7f and 0xff NaN;
// kAnyCode: +-480, in five instructions.
template <int F> __device__ __forceinline__ uint32_t code_word(uint32_t w) { return F == kInt8 ? w ^ 0x80808080u : w; }
template <int F, bool kAnyCode> __device__ __forceinline__ uint32_t code_pair(uint32_t w, bool upper) {
    if constexpr (F == kInt8) {
        return bits(__hsub2(as_h(__byte_perm(w, 0x64646464u, upper ? 0x4342 : 0x4140)), as_h(0x64806480u)));
    } else if constexpr (kAnyCode) {
        return bits(__hmul2(as_h(Decoder<__half, kE4m3>::fields(w, upper ? 2 : 0, upper ? 3 : 1)), as_h(0x5c005c00u)));
    } else {
        uint32_t r;
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(upper ? w >> 16 : w));
        return r;
    }
}

// 16 codes -> 16 values of T in two 16-byte vectors (lo: codes 0-7, hi: 8-15).
template <typename De>
__device__ __forceinline__ void decode16(const uint4& c, const De& d, uint4& lo, uint4& hi) {
    const uint32_t x = De::word(c.x), y = De::word(c.y), z = De::word(c.z), w = De::word(c.w);
    lo = make_uint4(d.pair(x, 0, 1), d.pair(x, 2, 3), d.pair(y, 0, 1), d.pair(y, 2, 3));
    hi = make_uint4(d.pair(z, 0, 1), d.pair(z, 2, 3), d.pair(w, 0, 1), d.pair(w, 2, 3));
}

// ---- write --------------------------------------------------------------------------------------
struct WriteArgs {
    const void* q;               // unused by the raw form
    const void* k;
    const void* v;
    const int32_t* mask;         // NULL in the raw form
    const int32_t* idx;          // NULL: row m is token m
    const int32_t* count;        // NULL: host_count
    int32_t host_count;
    const int32_t* pos;
    const float* norm_q;
    const float* norm_k;
    void* qc;
    uint8_t* save;               // per compact row: K codes, V codes, K scales, V scales of mask==1 rows
    int64_t ld_save;             // bytes
    Cache c;
    int64_t ld_qkv, ld_qc;
    int32_t n_tokens, n_heads, n_axes;
    float eps;
    float2 turns[kPairs];        // revolutions per position of each rotary pair, as a sum of two floats; 0: not rotated
    int8_t axis[kPairs];
};

// cos and sin of a rotary pair at position `pos`: the angle in revolutions, pos * turns, keeps its
// fraction to ~2^-30 for every position up to 2^24 (the product's rounding error is recovered by an
// fma), where a product in radians is off by pos * 2^-25. The codes are worth that: a K' near the
// border of two codes moves by a whole step.
__device__ __forceinline__ void rope_turn(float pos, float2 turns, float* sn, float* cs) {
    const float t = pos * turns.x;
    const float err = fmaf(pos, turns.x, -t);
    const float frac = (t - rintf(t)) + fmaf(pos, turns.y, err);
    sincospif(2.f * frac, sn, cs);
}

constexpr int kWriteThreads = 256;
constexpr int kWriteWarps = kWriteThreads / 32;
constexpr int kVecLanes = 8;                         // lanes of a head vector
constexpr int kVecHeads = 32 / kVecLanes;            // heads that a warp works on at a time
constexpr int kVecPairs = kHeadDim / kVecLanes / 2;  // element pairs of a lane

// A lane's 16 elements of a head vector in 32 bits.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4* x, float2* y) {
    const uint32_t u[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
    for (int t = 0; t < kVecPairs; ++t) y[t] = StoreT<T>::unpack2(u[t]);
}

// RMSNorm (w: the lane's weights) + RoPE.
__device__ __forceinline__ void norm_rope16(float2* y, const float2* w, float eps, const float* cs, const float* sn) {
    float2 s2 = f2mul(y[0], y[0]);
#pragma unroll
    for (int t = 1; t < kVecPairs; ++t) s2 = f2fma(y[t], y[t], s2);
    float ss = s2.x + s2.y;
#pragma unroll
    for (int o = kVecLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * (1.0f / kHeadDim) + eps);
#pragma unroll
    for (int t = 0; t < kVecPairs; ++t) {
        const float2 ab = f2mul(f2mul(y[t], make_float2(r, r)), w[t]);
        y[t] = make_float2(ab.x * cs[t] - ab.y * sn[t], ab.y * cs[t] + ab.x * sn[t]);
    }
}

// Quantises a head vector over its lanes and stores its codes and scale.
template <typename T, int F, bool kExact>
__device__ __forceinline__ void quantise_store(float2* y, uint8_t* codes, T* scale, int sub, bool active) {
    float m[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = max2n(fabsf(y[e].x), fabsf(y[e].y));
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = max3n(m[e], fabsf(y[4 + e].x), fabsf(y[4 + e].y));
    float amax = max2n(max3n(m[0], m[1], m[2]), m[3]);
#pragma unroll
    for (int o = kVecLanes / 2; o > 0; o >>= 1) amax = max2n(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float s = scale_of<T, F>(amax);
    // scales whose inverse is not a normal number are brought into range exactly; none: codes 0
    const bool tiny = s < 0x1p-100f, none = !(s > 0.f), capped = s >= scale_cap<T, F>();
    float r = __frcp_rn(s);
    uint4 w;
    if (__any_sync(0xffffffffu, tiny || none || capped)) {
        const float up = none ? 0.f : tiny ? 0x1p+100f : 1.f;
        r = none ? 0.f : __frcp_rn(s * up);
#pragma unroll
        for (int t = 0; t < kVecPairs; ++t)
            y[t] = none ? make_float2(0.f, 0.f) : make_float2(y[t].x * up, y[t].y * up);
        w = make_uint4(encode4<F, kExact>(y[0], y[1], r, true), encode4<F, kExact>(y[2], y[3], r, true),
                       encode4<F, kExact>(y[4], y[5], r, true), encode4<F, kExact>(y[6], y[7], r, true));
    } else {
        w = make_uint4(encode4<F, kExact>(y[0], y[1], r, false), encode4<F, kExact>(y[2], y[3], r, false),
                       encode4<F, kExact>(y[4], y[5], r, false), encode4<F, kExact>(y[6], y[7], r, false));
    }
    if (active) {
        *reinterpret_cast<uint4*>(codes + 16 * sub) = w;
        if (sub == 0) *reinterpret_cast<uint16_t*>(scale) = (uint16_t)StoreT<T>::pack2(s, s);
    }
}

// Executed rows into the 8-bit cache. Eight lanes hold a 128-wide head vector, 16 values each, so that
// rotary pairs are lane-local and the sum of squares and the largest magnitude are 3-step shuffles; a
// warp runs four heads of Q, K and V at a time (a unit). The launch's units are divided evenly over the
// warps, and a warp loads its next unit, also the next row's, while it works on one (1536 rows of 24 heads
// 13.6 us; 16.5 with a warp per row, which leaves a third of them idle, 17.1 with three per row). Three
// rows of T are read, one of T and two of bytes written per token (16896 rows of 24 heads in a graph: 101 us,
// 5.2 TB/s, with issue slots 62 % and DRAM 56 % busy; two lanes' worth of shuffles and a division per code
// took 211 us).
template <typename T, int F, bool kRaw>
__global__ void __launch_bounds__(kWriteThreads, 2) q8_write_kernel(const __grid_constant__ WriteArgs a) {
    const int lane = threadIdx.x & 31, sub = lane & (kVecLanes - 1), of = lane / kVecLanes;
    const int32_t warp = blockIdx.x * kWriteWarps + (threadIdx.x >> 5), warps = gridDim.x * kWriteWarps;
    pdl_launch_dependents();
    pdl_wait();
    const int32_t m_all = min(a.count ? *a.count : a.host_count, a.n_tokens);
    // the launch's line of (row, quad of heads) units, one range per warp
    const int32_t quads = (a.n_heads + kVecHeads - 1) / kVecHeads;
    const int64_t total = (int64_t)max(m_all, 0) * quads, per = max((int64_t)1, (total + warps - 1) / warps);
    const int64_t first = warp * per;
    int32_t left = (int32_t)(min(total, first + per) - first);
    if (left <= 0) return;
    float2 wq[kVecPairs], wk[kVecPairs];
    if (!kRaw) {
#pragma unroll
        for (int t = 0; t < kVecPairs; ++t) {
            const int e = 2 * (kVecPairs * sub + t);
            wq[t] = make_float2(a.norm_q[e], a.norm_q[e + 1]);
            wk[t] = make_float2(a.norm_k[e], a.norm_k[e + 1]);
        }
    }
    int32_t m = (int32_t)(first / quads), quad = (int32_t)(first - (int64_t)m * quads);
    auto token = [&](int32_t row) { return row < m_all ? (a.idx ? a.idx[row] : row) : -1; };
    auto listed = [&](int32_t i) { return i >= 0 && i < a.n_tokens; };
    uint4 nq[2], nk[2], nv[2];      // the next heads' vectors are on their way while these are worked on
    auto load = [&](int32_t i, int32_t quad) {
        const int32_t h = kVecHeads * quad + of;
        const int64_t at = (int64_t)i * a.ld_qkv + (int64_t)(h < a.n_heads ? h : 0) * kHeadDim + 16 * sub;
        const uint4* k = reinterpret_cast<const uint4*>(static_cast<const T*>(a.k) + at);
        const uint4* v = reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + at);
        if (!kRaw) {
            const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + at);
            nq[0] = __ldcs(q);
            nq[1] = __ldcs(q + 1);
        }
        nk[0] = __ldcs(k);
        nk[1] = __ldcs(k + 1);
        nv[0] = __ldcs(v);
        nv[1] = __ldcs(v + 1);
    };
    float cs[kVecPairs], sn[kVecPairs];
    int32_t i = token(m), next_i = -1;
    bool fresh = true, keep = false;
    if (listed(i)) load(i, quad);
    for (; left > 0; --left) {
        if (fresh) {
            fresh = false;
            next_i = token(m + 1);
            if (listed(i)) {
                keep = !kRaw && a.save != nullptr && a.mask[i] == 1;
                if (!kRaw) {
#pragma unroll
                    for (int t = 0; t < kVecPairs; ++t) {
                        const int j = kVecPairs * sub + t;
                        const float at = a.n_axes > 0 ? (float)a.pos[(int64_t)i * a.n_axes + a.axis[j]] : 0.f;
                        rope_turn(at, a.turns[j], &sn[t], &cs[t]);
                    }
                }
            } else if (lane == 0) {
                atomicOr(&g_error_word, kErrBounds);
            }
        }
        const bool last = quad + 1 == quads;
        const int32_t then_i = last ? next_i : i, then_quad = last ? 0 : quad + 1;
        if (listed(i)) {
            const int32_t h = kVecHeads * quad + of;
            const bool active = h < a.n_heads;
            const int64_t col = (int64_t)(active ? h : 0) * kHeadDim;
            uint8_t* ck = a.c.k + (int64_t)i * a.c.ld + col;
            uint8_t* cv = a.c.v + (int64_t)i * a.c.ld + col;
            T* ks = static_cast<T*>(a.c.ks) + (int64_t)(active ? h : 0) * a.c.ld_scale + i;
            T* vs = static_cast<T*>(a.c.vs) + (int64_t)(active ? h : 0) * a.c.ld_scale + i;
            if (keep && active) {
                uint8_t* sv = a.save + (int64_t)m * a.ld_save;
                const int64_t C = (int64_t)a.n_heads * kHeadDim;
                *reinterpret_cast<uint4*>(sv + col + 16 * sub) = *reinterpret_cast<const uint4*>(ck + 16 * sub);
                *reinterpret_cast<uint4*>(sv + C + col + 16 * sub) = *reinterpret_cast<const uint4*>(cv + 16 * sub);
                if (sub == 0) {
                    T* ss = reinterpret_cast<T*>(sv + 2 * C);
                    ss[h] = *ks;
                    ss[a.n_heads + h] = *vs;
                }
            }
            float2 y[kVecPairs];
            if (!kRaw) {
                unpack16<T>(nq, y);
                norm_rope16(y, wq, a.eps, cs, sn);
                if (active) {
                    uint4* q = reinterpret_cast<uint4*>(static_cast<T*>(a.qc) + (int64_t)m * a.ld_qc + col + 16 * sub);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        q[e] = make_uint4(StoreT<T>::pack2(y[4 * e].x, y[4 * e].y), StoreT<T>::pack2(y[4 * e + 1].x, y[4 * e + 1].y),
                                          StoreT<T>::pack2(y[4 * e + 2].x, y[4 * e + 2].y),
                                          StoreT<T>::pack2(y[4 * e + 3].x, y[4 * e + 3].y));
                }
            }
            unpack16<T>(nk, y);
            const uint4 xv[2] = {nv[0], nv[1]};
            if (left > 1 && listed(then_i)) load(then_i, then_quad);
            if (!kRaw) norm_rope16(y, wk, a.eps, cs, sn);
            quantise_store<T, F, kRaw>(y, ck, ks, sub, active);
            unpack16<T>(xv, y);
            quantise_store<T, F, true>(y, cv, vs, sub, active);
        } else if (left > 1 && listed(then_i)) {
            load(then_i, then_quad);
        }
        i = then_i;
        quad = then_quad;
        m += last;
        fresh = last;
    }
}

// ---- read ---------------------------------------------------------------------------------------
struct ReadArgs {
    Cache c;
    const int32_t* idx;          // NULL: output row m is cache row m
    const int32_t* count;        // NULL: host_count
    int32_t host_count;
    void* k;
    void* v;
    int64_t ld;
    int32_t n_rows, bound, n_heads;   // bound: rows that k and v hold, at most n_rows
};

constexpr int kReadThreads = 256;

// Rows back in T: each thread turns 16 codes (16 bytes) into two 16-byte vectors. Bound by memory.
template <typename T, int F>
__global__ void __launch_bounds__(kReadThreads) q8_read_kernel(const __grid_constant__ ReadArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int32_t asked = min(a.count ? *a.count : a.host_count, a.n_rows), m_all = min(asked, a.bound);
    if (asked > a.bound && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(&g_error_word, kErrBounds);
    const uint32_t per_row = (uint32_t)a.n_heads * (kHeadDim / 16);   // 16-code chunks of a row
    const int64_t total = (int64_t)m_all * per_row;
    const bool small = total <= 0xffffffffll;         // 32-bit divisions
    for (int64_t e = (int64_t)blockIdx.x * kReadThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kReadThreads) {
        const int32_t m = small ? (int32_t)((uint32_t)e / per_row) : (int32_t)(e / per_row);
        const int32_t c = (int32_t)(e - (int64_t)m * per_row);
        const int32_t i = a.idx ? a.idx[m] : m;
        if (i < 0 || i >= a.n_rows) {
            if (c == 0) atomicOr(&g_error_word, kErrBounds);
            continue;
        }
        const int64_t src = (int64_t)i * a.c.ld + c * 16, at = (int64_t)(c >> 3) * a.c.ld_scale + i;
        const int64_t dst = (int64_t)m * a.ld + c * 16;
        const uint4 ck = __ldcs(reinterpret_cast<const uint4*>(a.c.k + src));
        const uint4 cv = __ldcs(reinterpret_cast<const uint4*>(a.c.v + src));
        Decoder<T, F> dk, dv;
        dk.scale(0x10001u * static_cast<const uint16_t*>(a.c.ks)[at]);
        dv.scale(0x10001u * static_cast<const uint16_t*>(a.c.vs)[at]);
        uint4 lo, hi;
        decode16(ck, dk, lo, hi);
        uint4* ko = reinterpret_cast<uint4*>(static_cast<T*>(a.k) + dst);
        __stcs(ko, lo);
        __stcs(ko + 1, hi);
        decode16(cv, dv, lo, hi);
        uint4* vo = reinterpret_cast<uint4*>(static_cast<T*>(a.v) + dst);
        __stcs(vo, lo);
        __stcs(vo + 1, hi);
    }
}

// Rows of every stream's cache in T, packed [n_streams][n_tokens][n_heads * 128], for the 16-bit
// attention. There every row of a stream sees every key, so that a key whose K or V scale is not valid
// makes the head's rows NaN: its V row is NaN (and NaN times any weight), its K row zeros, since the
// 16-bit kernel's maximum and exponential may pass over a NaN score. The kernel also sets what the
// attention's launch needs: row counts that the bound holds, and zeroed arrivals. Bound by memory.
struct ExpandArgs {
    Cache src[kMaxBatch];
    const int32_t* count[kMaxBatch];
    int32_t n_streams, n_tokens, n_heads, max_rows;
    void* k;
    void* v;
    int32_t* rows;               // [n_streams] counts, clamped to max_rows
    uint4* zero;
    int32_t n_zero;
};

template <typename T, int F>
__global__ void __launch_bounds__(kReadThreads) q8_expand_kernel(const __grid_constant__ ExpandArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t first = (int64_t)blockIdx.x * kReadThreads + threadIdx.x, stride = (int64_t)gridDim.x * kReadThreads;
    if (blockIdx.x == 0 && threadIdx.x < kMaxBatch) {
#pragma unroll
        for (int b = 0; b < kMaxBatch; ++b)
            if (b == (int)threadIdx.x && b < a.n_streams) {
                const int32_t m = *a.count[b];
                if (m > a.max_rows) atomicOr(&g_error_word, kErrBounds);
                a.rows[b] = max(0, min(m, a.max_rows));
            }
    }
    for (int64_t e = first; e < a.n_zero; e += stride) a.zero[e] = make_uint4(0, 0, 0, 0);
    const uint32_t per_row = (uint32_t)a.n_heads * (kHeadDim / 16);
    const int64_t total = (int64_t)a.n_tokens * per_row;
    const bool small = total <= 0xffffffffll;
    const Cache c = a.src[blockIdx.y];
    T* ko = static_cast<T*>(a.k) + blockIdx.y * total * 16;
    T* vo = static_cast<T*>(a.v) + blockIdx.y * total * 16;
    for (int64_t e = first; e < total; e += stride) {
        const int32_t i = small ? (int32_t)((uint32_t)e / per_row) : (int32_t)(e / per_row);
        const int32_t h16 = (int32_t)(e - (int64_t)i * per_row);
        const uint4 ck = __ldcs(reinterpret_cast<const uint4*>(c.k + i * c.ld + h16 * 16));
        const uint4 cv = __ldcs(reinterpret_cast<const uint4*>(c.v + i * c.ld + h16 * 16));
        const int64_t at = (int64_t)(h16 >> 3) * c.ld_scale + i;
        uint32_t sk = static_cast<const uint16_t*>(c.ks)[at], sv = static_cast<const uint16_t*>(c.vs)[at];
        const bool ok = valid_scale<T, F>(StoreT<T>::unpack2(sk).x) && valid_scale<T, F>(StoreT<T>::unpack2(sv).x);
        if (!ok) sk = 0;
        typename TileDecoder<T, F>::any dk, dv;
        dk.scale(0x10001u * sk);
        dv.scale(0x10001u * sv);
        uint4 lo, hi;
        decode16(ck, dk, lo, hi);
        uint4* o = reinterpret_cast<uint4*>(ko + e * 16);
        o[0] = lo;
        o[1] = hi;
        decode16(cv, dv, lo, hi);
        if (!ok) lo = hi = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);   // NaN of either type
        o = reinterpret_cast<uint4*>(vo + e * 16);
        o[0] = lo;
        o[1] = hi;
    }
}

// ---- restore ------------------------------------------------------------------------------------
struct RestoreArgs {
    Cache c;
    const int32_t* mask;
    const int32_t* idx;
    const int32_t* count;
    const uint8_t* save;
    int64_t ld_save;
    int32_t n_tokens, n_heads;
};

// Codes and scales of mask==1 rows back from `save`: a warp per executed row, which leaves at once
// where the row keeps its new codes.
__global__ void __launch_bounds__(256) q8_restore_kernel(const __grid_constant__ RestoreArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int32_t m_all = min(*a.count, a.n_tokens);
    const int64_t C = (int64_t)a.n_heads * kHeadDim;
    for (int32_t m = blockIdx.x * 8 + (threadIdx.x >> 5); m < m_all; m += gridDim.x * 8) {
        const int32_t i = a.idx[m];
        if (i < 0 || i >= a.n_tokens || a.mask[i] != 1) continue;   // a bad index: flagged by the write
        const uint8_t* sv = a.save + (int64_t)m * a.ld_save;
        for (int64_t e = lane * 16; e < C; e += 32 * 16) {
            *reinterpret_cast<uint4*>(a.c.k + (int64_t)i * a.c.ld + e) = *reinterpret_cast<const uint4*>(sv + e);
            *reinterpret_cast<uint4*>(a.c.v + (int64_t)i * a.c.ld + e) = *reinterpret_cast<const uint4*>(sv + C + e);
        }
        const uint16_t* ss = reinterpret_cast<const uint16_t*>(sv + 2 * C);
        for (int32_t h = lane; h < a.n_heads; h += 32) {
            static_cast<uint16_t*>(a.c.ks)[(int64_t)h * a.c.ld_scale + i] = ss[h];
            static_cast<uint16_t*>(a.c.vs)[(int64_t)h * a.c.ld_scale + i] = ss[a.n_heads + h];
        }
    }
}

}  // namespace q8
}  // namespace fxr
