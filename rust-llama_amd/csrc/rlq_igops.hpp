// rlq_igops.hpp - the weight operands of the int8 products (igemm.hip, moe.hip):
// every weight format's int8 planes of scale times level, made in registers from
// the packed weights of the tiled layout (rlq_layout.hpp), for
// v_mfma_i32_32x32x32_i8.
#pragma once

#include <type_traits>

#include "rlq_device.hpp"
#include "rlq_internal.hpp"
#include "rlq_layout.hpp"

namespace rlq {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__host__ __device__ constexpr bool ig_mins(uint32_t t) { return t == kQ2_K || t == kQ4_K || t == kQ5_K; }
__host__ __device__ constexpr bool ig_slots(uint32_t t) { return t == kQ4_K || t == kQ5_K; }

// ---------------------------------------------------------------------------
// Weight operands
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint4 ig_ld16(const uint8_t* p) { return *(const uint4*)p; }
__device__ __forceinline__ uint32_t ig_word(const uint4& v, int i) {
    return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w));
}
__device__ __forceinline__ uint32_t pk_mul(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, (u16x2)(__builtin_bit_cast(u16x2, a) * __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t pk_mad(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_bit_cast(
        uint32_t, (u16x2)(__builtin_bit_cast(u16x2, a) * __builtin_bit_cast(u16x2, b) + __builtin_bit_cast(u16x2, c)));
}
// Byte B of w in both 16-bit halves, zero- or sign-extended.
template <int B>
__device__ __forceinline__ uint32_t ubyte2(uint32_t w) {
    return __builtin_amdgcn_perm(0u, w, 0x0c000c00u | (uint32_t)B | (uint32_t)B << 16);
}
__device__ __forceinline__ uint32_t pair16(int32_t v) { return (uint32_t)(uint16_t)v | (uint32_t)v << 16; }

// p + 128 of four values (even and odd bytes as 16-bit pairs) -> the two planes
// of p: the high byte, and the low byte with its top bit flipped (p + 128 =
// 256 hi + (lo + 128)).
__device__ __forceinline__ void split_planes(uint32_t e, uint32_t o, int32_t& hi, int32_t& lo) {
    hi = (int32_t)__builtin_amdgcn_perm(o, e, 0x07030501u);
    lo = (int32_t)(__builtin_amdgcn_perm(o, e, 0x06020400u) ^ 0x80808080u);
}

// A 4-bit field of eight mins or scales (bytes of two words) as f16: 0x64kk is
// 1024 + kk.
__device__ __forceinline__ f16x2 ig_byte_half2(uint32_t w, uint32_t sel) {
    return __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)) -
           (f16x2){(_Float16)1024.0f, (_Float16)1024.0f};
}

// One format: Raw holds a lane's loaded bytes of one (16-row tile, chunk) pair:
// head loads the scales, refill<S> the pieces that no k-step after S uses (kLoads
// of them in 16 bytes each, not next to each other); Pre is
// what a chunk's k-steps share; ops<S> makes the weight operand of k-step S.
// Lane (ln, kh) of a wave works on row ln % 16 = n of layout tile ln / 16 and k
// half kh.
template <uint32_t T>
struct Ig;

template <>
struct Ig<kQ2_K> {
    static constexpr uint32_t kChunk = kQ2KChunk;
    static constexpr int kLoads = 3;
    static constexpr int kPlanes = 1, kShift = 0;
    struct Raw {
        uint4 q[2], sc;
        uint32_t dd;
    };
    struct Pre {
        uint32_t c[4];
    };
    __device__ static void head(Raw& r, const uint8_t* p, uint32_t n) {
        r.sc = ig_ld16(p + 1024 + n * 16);
        r.dd = *(const uint32_t*)(p + 1280 + n * 4);
    }
    template <int S>
    __device__ static void refill(Raw& r, const uint8_t* p, uint32_t n, uint32_t kh) {
        if (S % 4 == 3) r.q[S / 4] = ig_ld16(p + (16 * (2 * (S / 4) + kh) + n) * 16);
    }
    __device__ static Pre pre(const Raw& r, uint32_t kh) {
        Pre o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o.c[k] = (ig_word(r.sc, k) >> (8 * kh)) & 0x000f000fu;
        return o;
    }
    // scale index 8 (S / 4) + 2 (S % 4) + kh: word S / 2, half S % 2 of the shifted words
    template <int S>
    __device__ static void ops(const Raw& r, const Pre& c, i32x4& a, i32x4&) {
        const uint32_t w = c.c[S / 2];
        const uint32_t sc = __builtin_amdgcn_perm(0u, w, (S & 1) ? 0x03020302u : 0x01000100u);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            a[i] = (int32_t)pk_mul((ig_word(r.q[S / 4], i) >> (2 * (S % 4))) & 0x03030303u, sc);
    }
    __device__ static f16x8 mins(const Raw& r, uint32_t kh) {
        const uint32_t w0 = ((kh ? r.sc.z : r.sc.x) >> 4) & 0x0f0f0f0fu, w1 = ((kh ? r.sc.w : r.sc.y) >> 4) & 0x0f0f0f0fu;
        f16x8 m;
        const f16x2 a = ig_byte_half2(w0, 0x04010400u), b = ig_byte_half2(w0, 0x04030402u);
        const f16x2 c = ig_byte_half2(w1, 0x04010400u), d = ig_byte_half2(w1, 0x04030402u);
        m[0] = a[0], m[1] = a[1], m[2] = b[0], m[3] = b[1], m[4] = c[0], m[5] = c[1], m[6] = d[0], m[7] = d[1];
        return m;
    }
    __device__ static float d(const Raw& r) { return half_to_float(r.dd); }
    __device__ static float dmin(const Raw& r) { return half_to_float(r.dd >> 16); }
};

template <>
struct Ig<kQ3_K> {
    static constexpr uint32_t kChunk = kQ3KChunk;
    static constexpr int kLoads = 3;
    static constexpr int kPlanes = 1, kShift = 0;
    struct Raw {
        uint4 q[2], hm;
        uint32_t s0, s1, s2, d;
    };
    struct Pre {
        uint32_t c[4];
    };
    template <int S>
    __device__ static void refill(Raw& r, const uint8_t* p, uint32_t n, uint32_t kh) {
        if (S % 4 == 3) r.q[S / 4] = ig_ld16(p + (16 * (2 * (S / 4) + kh) + n) * 16);
        if (S == 7) r.hm = ig_ld16(p + 1024 + n * 32 + 16 * kh);
    }
    __device__ static void head(Raw& r, const uint8_t* p, uint32_t n) {
        const uint32_t* s = (const uint32_t*)(p + 1536 + n * 12);
        r.s0 = s[0], r.s1 = s[1], r.s2 = s[2];
        r.d = *(const uint16_t*)(p + 1728 + n * 2);
    }
    __device__ static Pre pre(const Raw& r, uint32_t kh) {
        // 6-bit scales (matvec_extra.rs:200-210), 0..63 for -32..31
        Pre o;
        o.c[0] = (r.s0 & 0x0f0f0f0fu) | ((r.s2 << 4) & 0x30303030u);
        o.c[1] = (r.s1 & 0x0f0f0f0fu) | ((r.s2 << 2) & 0x30303030u);
        o.c[2] = ((r.s0 >> 4) & 0x0f0f0f0fu) | (r.s2 & 0x30303030u);
        o.c[3] = ((r.s1 >> 4) & 0x0f0f0f0fu) | ((r.s2 >> 2) & 0x30303030u);
#pragma unroll
        for (int k = 0; k < 4; ++k) o.c[k] = (o.c[k] >> (8 * kh)) & 0x003f003fu;
        return o;
    }
    // -(sc * (u - 4)) mod 256 with u = 0..7: u * (32 - s) + 4 (s - 32)
    template <int S>
    __device__ static void ops(const Raw& r, const Pre& c, i32x4& a, i32x4&) {
        const uint32_t s = __builtin_amdgcn_perm(0u, c.c[S / 2], (S & 1) ? 0x03020302u : 0x01000100u);
        const uint32_t neg = __builtin_bit_cast(uint32_t, (u16x2)((u16x2){32, 32} - __builtin_bit_cast(u16x2, s)));
        const uint32_t add = __builtin_bit_cast(uint32_t, (u16x2)(__builtin_bit_cast(u16x2, neg) * (u16x2){0xfffc, 0xfffc}));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t low = (ig_word(r.q[S / 4], i) >> (2 * (S % 4))) & 0x03030303u;
            const uint32_t h = ig_word(r.hm, i);
            const uint32_t u = low | ((S < 2 ? h << (2 - S) : h >> (S - 2)) & 0x04040404u);
            const uint32_t e = pk_mad(u & 0x00ff00ffu, neg, add), o = pk_mad((u >> 8) & 0x00ff00ffu, neg, add);
            a[i] = (int32_t)__builtin_amdgcn_perm(o, e, 0x06020400u);
        }
    }
    __device__ static float d(const Raw& r) { return -half_to_float(r.d); }
};

// Q4_K / Q5_K header words: 6-bit scales and mins (get_scale_min_k4,
// crates/quant/src/decode.rs:216-235), four per word.
struct IgHead {
    uint32_t scA, scB, mnA, mnB;
};
__device__ __forceinline__ IgHead ig_head(const uint4& h) {
    IgHead q;
    q.scA = h.y & 0x3f3f3f3fu;
    q.scB = (h.w & 0x0f0f0f0fu) | ((h.y >> 2) & 0x30303030u);
    q.mnA = h.z & 0x3f3f3f3fu;
    q.mnB = ((h.w >> 4) & 0x0f0f0f0fu) | ((h.z >> 2) & 0x30303030u);
    return q;
}
// mins of sub-blocks 4 kh .. 4 kh + 3, each against two 16-value sums
__device__ __forceinline__ f16x8 ig_head_mins(const uint4& h, uint32_t kh) {
    const IgHead q = ig_head(h);
    const uint32_t w = kh ? q.mnB : q.mnA;
    f16x8 m;
    const f16x2 a = ig_byte_half2(w, 0x04010400u), b = ig_byte_half2(w, 0x04030402u);
    m[0] = m[1] = a[0], m[2] = m[3] = a[1], m[4] = m[5] = b[0], m[6] = m[7] = b[1];
    return m;
}

template <>
struct Ig<kQ4_K> {
    static constexpr uint32_t kChunk = kQ4KChunk;
    static constexpr int kLoads = 5;
    static constexpr int kPlanes = 2, kShift = 3;
    struct Raw {
        uint4 q[4], h;
    };
    struct Pre {
        uint32_t hi[2], lo[2];
    };
    __device__ static void head(Raw& r, const uint8_t* p, uint32_t n) { r.h = ig_ld16(p + 2048 + n * 16); }
    template <int S>
    __device__ static void refill(Raw& r, const uint8_t* p, uint32_t n, uint32_t kh) {
        if (S & 1) r.q[S / 2] = ig_ld16(p + (S / 4) * 1024 + (16 * (2 * (S / 2 % 2) + kh) + n) * 16);
    }
    __device__ static Pre pre(const Raw& r, uint32_t) {
        const IgHead q = ig_head(r.h);
        return Pre{{(q.scA >> 3) & 0x07070707u, (q.scB >> 3) & 0x07070707u}, {q.scA & 0x07070707u, q.scB & 0x07070707u}};
    }
    template <int S>
    __device__ static void ops(const Raw& r, const Pre& c, i32x4& a, i32x4& b) {
        const uint32_t sh = ubyte2<S % 4>(c.hi[S / 4]), sl = ubyte2<S % 4>(c.lo[S / 4]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = ig_word(r.q[S / 2], i), q = ((S & 1) ? w >> 4 : w) & 0x0f0f0f0fu;
            a[i] = (int32_t)pk_mul(q, sh);  // byte products <= 105: no carries between bytes
            b[i] = (int32_t)pk_mul(q, sl);
        }
    }
    __device__ static f16x8 mins(const Raw& r, uint32_t kh) { return ig_head_mins(r.h, kh); }
    __device__ static float d(const Raw& r) { return half_to_float(r.h.x); }
    __device__ static float dmin(const Raw& r) { return half_to_float(r.h.x >> 16); }
};

template <>
struct Ig<kQ5_K> {
    static constexpr uint32_t kChunk = kQ5KChunk;
    static constexpr int kLoads = 6;
    static constexpr int kPlanes = 2, kShift = 8;
    struct Raw {
        uint4 q[4], qh, h;
    };
    struct Pre {
        uint32_t sc[2];
    };
    __device__ static void head(Raw& r, const uint8_t* p, uint32_t n) { r.h = ig_ld16(p + 2560 + n * 16); }
    template <int S>
    __device__ static void refill(Raw& r, const uint8_t* p, uint32_t n, uint32_t kh) {
        if (S & 1) r.q[S / 2] = ig_ld16(p + (S / 4) * 1024 + (16 * (2 * (S / 2 % 2) + kh) + n) * 16);
        if (S == 7) r.qh = ig_ld16(p + 2048 + n * 32 + 16 * kh);
    }
    __device__ static Pre pre(const Raw& r, uint32_t) {
        const IgHead q = ig_head(r.h);
        return Pre{{q.scA, q.scB}};
    }
    template <int S>
    __device__ static void ops(const Raw& r, const Pre& c, i32x4& a, i32x4& b) {
        const uint32_t sc = ubyte2<S % 4>(c.sc[S / 4]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = ig_word(r.q[S / 2], i), h = ig_word(r.qh, i);
            const uint32_t u = (((S & 1) ? w >> 4 : w) & 0x0f0f0f0fu) | ((S < 4 ? h << (4 - S) : h >> (S - 4)) & 0x10101010u);
            const uint32_t e = pk_mad(u & 0x00ff00ffu, sc, 0x00800080u), o = pk_mad((u >> 8) & 0x00ff00ffu, sc, 0x00800080u);
            int32_t hi, lo;
            split_planes(e, o, hi, lo);
            a[i] = hi, b[i] = lo;
        }
    }
    __device__ static f16x8 mins(const Raw& r, uint32_t kh) { return ig_head_mins(r.h, kh); }
    __device__ static float d(const Raw& r) { return half_to_float(r.h.x); }
    __device__ static float dmin(const Raw& r) { return half_to_float(r.h.x >> 16); }
};

template <>
struct Ig<kQ6_K> {
    static constexpr uint32_t kChunk = kQ6KChunk;
    static constexpr int kLoads = 7;
    static constexpr int kPlanes = 2, kShift = 8;
    struct Raw {
        uint4 ql[4], qh[2], sc;
        uint32_t d;
    };
    struct Pre {
        uint32_t c[4];
    };
    __device__ static void head(Raw& r, const uint8_t* p, uint32_t n) {
        r.sc = ig_ld16(p + 3072 + n * 16);
        r.d = *(const uint16_t*)(p + 3328 + n * 2);
    }
    template <int S>
    __device__ static void refill(Raw& r, const uint8_t* p, uint32_t n, uint32_t kh) {
        if (S % 4 >= 2) r.ql[2 * (S / 4) + S % 2] = ig_ld16(p + kh * 1024 + (16 * (2 * (S / 4) + S % 2) + n) * 16);
        if (S % 4 == 3) r.qh[S / 4] = ig_ld16(p + 2048 + n * 64 + 32 * (S / 4) + 16 * kh);
    }
    __device__ static Pre pre(const Raw& r, uint32_t kh) {
        Pre o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o.c[k] = ig_word(r.sc, k) >> (8 * kh);
        return o;
    }
    // k-step S = 4 (half of the block) + side; scale index 2 S + kh
    template <int S>
    __device__ static void ops(const Raw& r, const Pre& c, i32x4& a, i32x4& b) {
        constexpr int kSide = S % 4, kG = S / 4;
        const int32_t s = __builtin_amdgcn_sbfe((int32_t)c.c[S / 2], 16 * (S % 2), 8);
        const uint32_t sc = pair16(s), add = pair16(128 - 32 * s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = ig_word(r.ql[2 * kG + (kSide & 1)], i), h = ig_word(r.qh[kG], i);
            const uint32_t u = ((kSide < 2 ? w : w >> 4) & 0x0f0f0f0fu) |
                               ((kSide < 2 ? h << (4 - 2 * kSide) : h >> (2 * kSide - 4)) & 0x30303030u);
            const uint32_t e = pk_mad(u & 0x00ff00ffu, sc, add), o = pk_mad((u >> 8) & 0x00ff00ffu, sc, add);
            int32_t hi, lo;
            split_planes(e, o, hi, lo);
            a[i] = hi, b[i] = lo;
        }
    }
    __device__ static float d(const Raw& r) { return half_to_float(r.d); }
};

template <int S>
using IgStep = std::integral_constant<int, S>;
// f(IgStep<0>), ..., f(IgStep<7>)
template <typename F>
__device__ __forceinline__ void ig_steps(F&& f) {
    f(IgStep<0>{}), f(IgStep<1>{}), f(IgStep<2>{}), f(IgStep<3>{});
    f(IgStep<4>{}), f(IgStep<5>{}), f(IgStep<6>{}), f(IgStep<7>{});
}
template <uint32_t T>
__device__ __forceinline__ void ig_load(typename Ig<T>::Raw& r, const uint8_t* p, uint32_t n, uint32_t kh) {
    ig_steps([&](auto s) { Ig<T>::template refill<decltype(s)::value>(r, p, n, kh); });
    Ig<T>::head(r, p, n);
}

// Q8_0: a chunk of four layout pairs (eight blocks of 32)
template <uint32_t T>
struct IgRaw {
    using Raw = typename Ig<T>::Raw;
};
template <>
struct IgRaw<kQ8_0> {
    struct Raw {
        uint4 q[8];
        uint32_t d[4];
    };
};

__device__ __forceinline__ i32x16 ig_mfma(i32x4 a, i32x4 b, i32x16 c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

}  // namespace rlq
