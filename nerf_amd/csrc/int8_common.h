// Pieces shared by the 8-bit dense-layer kernels (int8_quantize.hip, int8_product.h, int8_linear.hip, int8_grad_input.hip,
// int8_grad_weight.hip): number formats, the layout of packed weights, loads and stores of rows of any type
// and alignment.
//
// Rows: q [n][kp] int8, kp = k rounded up to 64, zeros behind column k; one fp32 scale per row;
// optionally one bit per element (element > 0), bit f & 7 of byte f >> 3 of a row of kp / 8 bytes.
//
// Packed weights of W [k][m] (Keras [in, out]), mp = m rounded up to 64:
//   float scale[mp]                            one per output channel, 0 behind m
//   int8 fragments [mp/64][kp/64][4][64][16]   the integers, A operands of v_mfma_i32_16x16x64_i8
//   bf16 fragments [kp/64][mp/32][4][64][8]    only with power-of-two scales: integer x scale (exact in
//                                              bf16: 7 bits), A operands of v_mfma_f32_16x16x32_bf16
// A fragment is 1 KiB: lane = row (16 output features) + 16 x piece of the contraction (16 integers or
// 8 bf16).  Row r of fragment u of a group of 64 features is feature 16 (r >> 2) + 4 u + (r & 3) of
// the group: read as stored, a lane's accumulators (point = lane & 15, g = lane >> 4) over the four fragments
// are features 16 g .. 16 g + 15, what an 8-bit output stores; for wider types the products read the rows in
// the order that leaves a lane pieces of 16 bytes.
#pragma once
#include "common.h"

#define DEV __device__ __forceinline__

namespace nerf {
namespace i8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__host__ __device__ inline int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }

constexpr int kMaxWidth = 65536;  // |sum| <= 65536 x 127^2 < 2^31: the int32 sums cannot overflow

struct PackedLayout {
    int kp, mp;
    size_t frags, frags_t, bytes;
    __host__ __device__ PackedLayout(int k, int m, bool with_grad) {
        kp = (int)up64(k), mp = (int)up64(m);
        frags = (size_t)mp * 4;
        frags_t = frags + (size_t)mp * kp;
        bytes = frags_t + (with_grad ? (size_t)mp * kp * 2 : 0);
    }
};

// Feature (inside its group of 64) of row r of fragment u.
__host__ __device__ inline int frag_feature(int u, int r) { return 16 * (r >> 2) + 4 * u + (r & 3); }

// ---- element types --------------------------------------------------------------------------------
template <int DT> struct Elem;
template <> struct Elem<NERF_F32> { typedef float T; };
template <> struct Elem<NERF_F16> { typedef _Float16 T; };
template <> struct Elem<NERF_BF16> { typedef __bf16 T; };

inline bool dtype_ok(int dt) { return dt == NERF_F32 || dt == NERF_F16 || dt == NERF_BF16; }
inline int dtype_size(int dt) { return dt == NERF_F32 ? 4 : 2; }

// 16 bytes at any address that the element type allows (global memory takes unaligned vectors).
typedef int i32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef int i32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef int i32u __attribute__((aligned(2)));

// Eight neighbouring elements as they are loaded: one register quad of 16-bit elements, or two of fp32.
template <class T> struct Raw8 {
    i32x4 w[sizeof(T) / 2 == 1 ? 1 : 2];
};

template <class T>
DEV void to_float(const Raw8<T>& r, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int w = r.w[i >> 2][i & 3];  // (a bit cast of a vector's element itself takes element 0)
            v[i] = __builtin_bit_cast(float, w);
        }
    } else if constexpr (__is_same(T, __bf16)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __builtin_bit_cast(float, r.w[0][i] << 16);
            v[2 * i + 1] = __builtin_bit_cast(float, r.w[0][i] & (int)0xffff0000);
        }
    } else {
        typedef _Float16 half8 __attribute__((ext_vector_type(8)));
        const half8 h = __builtin_bit_cast(half8, r.w[0]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    }
}

// Elements c .. c + 7 of a row of `width`; those behind its end are zero.  `whole` (the same in every lane):
// no lane's piece passes the end.  A piece that does is read so that it ends with the row, and shifted
// down: three steps of selects instead of eight guarded loads.
template <class T>
DEV Raw8<T> load8(const T* row, int c, int width, bool whole) {
    Raw8<T> r;
    constexpr int W = sizeof(T) == 4 ? 8 : 4;  // words of a piece
    if (whole) {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) r.w[i] = *(const i32x4u*)((const char*)(row + c) + 16 * i);
        return r;
    }
    int w[W];
    if (width >= 8) {
        const int over = c + 8 - width;  // elements behind the end
        const T* src = row + (over > 0 ? width - 8 : c);
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const i32x4 q = *(const i32x4u*)((const char*)src + 16 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * i + j] = q[j];
        }
        const int e = over < 0 ? 0 : over;
        if constexpr (W == 8) {
#pragma unroll
            for (int k = 4; k >= 1; k /= 2)
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = (e & k) ? (i + k < 8 ? w[i + k] : 0) : w[i];
        } else {
#pragma unroll
            for (int k = 2; k >= 1; k /= 2)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = (e & (2 * k)) ? (i + k < 4 ? w[i + k] : 0) : w[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (e & 1) ? (int)((unsigned)w[i] >> 16 | (i < 3 ? (unsigned)w[i + 1] << 16 : 0u)) : w[i];
        }
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = e >= 8 ? 0 : w[i];
    } else {  // a row shorter than a piece
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (W == 8) {
                w[i] = c + i < width ? __builtin_bit_cast(int, row[c + i]) : 0;
            } else {
                const unsigned lo = c + 2 * i < width ? __builtin_bit_cast(unsigned short, row[c + 2 * i]) : 0;
                const unsigned hi = c + 2 * i + 1 < width ? __builtin_bit_cast(unsigned short, row[c + 2 * i + 1]) : 0;
                w[i] = (int)(lo | hi << 16);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i >> 2][i & 3] = w[i];
    return r;
}

// N consecutive elements at p (any alignment the element type allows) as floats; only the first `have`
// exist, the others read as zero.
template <class T, int N>
DEV void load_row(const T* p, int have, float (&v)[N]) {
    if (have >= N) {
        T t[N];
        __builtin_memcpy(t, p, sizeof t);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < have ? (float)p[i] : 0.f;
    }
}

// ---- scales ----------------------------------------------------------------------------------------
// Of a row or channel whose largest magnitude has the bit pattern `top` (a non-negative float orders like
// its bits; NaN sorts above infinity).  `scale` is what an integer stands for, `inv` what a value is
// multiplied by before it is rounded.
//  - power of two: the smallest 2^e >= top / 127, not below 2^-126: rounding is the only loss, and an
//    integer times its scale is exact in bf16, so that the gradients' products are exact;
//  - otherwise top / 127: on average 0.7 of the step of the power of two.  Below 2^-100, where the
//    inverse would overflow, the row is held as zeros;
//  - infinity or NaN in the row: the scale is NaN, the integers zero; every product of it is NaN.
struct Scale {
    float scale, inv;
};
DEV Scale scale_of(unsigned top, bool pow2) {
    if (top >= 0x7f800000u) return {__builtin_bit_cast(float, 0x7fc00000u), 0.f};
    if (pow2) {
        int e = (int)(top >> 23) - 133 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
        e = e < -126 ? -126 : e;
        return {__builtin_bit_cast(float, (unsigned)(e + 127) << 23), __builtin_bit_cast(float, (unsigned)(127 - e) << 23)};
    }
    if (top < (27u << 23)) return {0.f, 0.f};
    const float a = __builtin_bit_cast(float, top);
    return {a / 127.f, 127.f / a};
}
DEV unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }
// The integer of v: halves to even; a row without a sound scale (inv = 0) gives zeros, NaN included.
DEV int quantised(float v, float inv) { return inv == 0.f ? 0 : (int)__builtin_rintf(v * inv); }

DEV unsigned pack4(int a, int b, int c, int d) {
    return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)d << 24;
}

// Rounding to bytes, halves to even: a number of magnitude at most 127.5 added to 1.5 x 2^23, where a
// float's step is 1, leaves its integer in the low byte (one addition instead of a rounding and a
// conversion); four low bytes are gathered with byte permutations.
constexpr float kRoundAt = 12582912.f;
DEV unsigned low_bytes(const float (&t)[4]) {
    unsigned b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __builtin_bit_cast(unsigned, t[i]);
    const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// ---- bf16 terms -------------------------------------------------------------------------------------
// How many bf16 numbers a value of a type is the exact sum of (8, 11 and 24 bits of 8 each).
template <int DT> struct Terms { static constexpr int N = DT == NERF_BF16 ? 1 : DT == NERF_F16 ? 2 : 3; };

// v as the sum of N bf16 terms, each the leading bits (cut off, not rounded: a value near the fp32 maximum would
// round to infinity) of what the ones before it leave: exact down to bf16's smallest steps.  An infinity is its
// first term, with zeros behind; a NaN is one in the first or the second.
template <int N>
DEV void split_bf16(const float (&v)[8], bf16x8 (&t)[N]) {
    unsigned rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = __builtin_bit_cast(unsigned, v[i]);
#pragma unroll
    for (int s = 0; s < N; ++s) {
        i32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (int)__builtin_amdgcn_perm(rest[2 * i + 1], rest[2 * i], 0x07060302u);
        t[s] = __builtin_bit_cast(bf16x8, w);
        if (s + 1 < N) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float left = __builtin_bit_cast(float, rest[i]) - __builtin_bit_cast(float, rest[i] & 0xffff0000u);
                const bool inf = s == 0 && __builtin_fabsf(v[i]) == __builtin_inff();
                rest[i] = inf ? 0u : __builtin_bit_cast(unsigned, left);
            }
        }
    }
}

}  // namespace i8
}  // namespace nerf
