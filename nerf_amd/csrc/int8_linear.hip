// Products of rows with packed weights: nerf_linear_int8 (8-bit integers, int32 sums) and
// nerf_linear_int8_grad_input (bf16 terms, fp32 sums).  Formats: int8_common.h.
//
// Both are D[feature][point] = sum over the contraction of A[feature][c] B[c][point] with 16 x 16 tiles:
// A fragments are stored as the matrix unit takes them, a lane's B fragment is 16 integers (8 bf16)
// that lie next to each other in its point's row, and the four tiles of a group of 64 features leave
// 16 neighbouring features of one point in a lane.
#include "int8_common.h"

namespace nerf {
namespace i8 {

struct LinearArgs {
    const char* frags;     // this product's fragments
    int groups, steps;     // groups of 64 features, steps of 64 integers (32 bf16)
    int64_t n;
    // the rows: q and scale, or dz
    const signed char* q;
    const float* scale;
    const void* dz;
    int64_t lddz;
    int width;             // columns of dz (the contraction)
    // what becomes of the sums
    int features;          // of a row of the output
    const float* wscale;
    const float* bias;
    const void* addend;    // [n][ldadd] or null
    int add_dtype;
    int64_t ldadd;
    int relu;
    const unsigned char* mask;
    void* out;
    int64_t ldout;
};

// ---- the two products -----------------------------------------------------------------------------
struct Int8Op {
    typedef i32x4 Acc;
    struct B {
        i32x4 v;
    };
    static DEV Acc zero() { return Acc{0, 0, 0, 0}; }
    static DEV B load(const LinearArgs& a, int64_t p, int s, int g) {
        return {*(const i32x4*)(a.q + (p * a.steps + s) * 64 + 16 * g)};
    }
    static DEV Acc mma(i32x4 w, const B& b, Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, b.v, c, 0, 0, 0); }
};

template <int DT>
struct Bf16Op {
    typedef f32x4 Acc;
    static constexpr int N = Terms<DT>::N;
    struct B {
        bf16x8 v[N];
    };
    static DEV Acc zero() { return Acc{0.f, 0.f, 0.f, 0.f}; }
    static DEV B load(const LinearArgs& a, int64_t p, int s, int g) {
        typedef typename Elem<DT>::T T;
        const int c = 32 * s + 8 * g;
        const T* src = (const T*)a.dz + p * a.lddz + c;
        B b;
        if constexpr (DT == NERF_BF16) {
            if (c + 8 <= a.width) {
                __builtin_memcpy(&b.v[0], src, 16);
                return b;
            }
        }
        float v[8];
        load_row<T, 8>(src, a.width - c, v);
        split_bf16<N>(v, b.v);
        return b;
    }
    static DEV Acc mma(i32x4 w, const B& b, Acc c) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), b.v[i], c, 0, 0, 0);
        return c;
    }
};

// ---- what becomes of the sums of a lane: 16 neighbouring features of point p -------------------------
DEV void load16(const void* p, int dtype, int64_t at, int have, float (&v)[16]) {
    if (dtype == NERF_F32) load_row<float, 16>((const float*)p + at, have, v);
    else if (dtype == NERF_F16) load_row<_Float16, 16>((const _Float16*)p + at, have, v);
    else load_row<__bf16, 16>((const __bf16*)p + at, have, v);
}

// y = relu((sum x channel scale) x row scale + bias + addend), each step rounded to fp32, then to the
// output's type.
DEV void finish_linear(const LinearArgs& a, const i32x4 (&acc)[4], int T, int64_t p, int g, float (&v)[16]) {
    const int f = 64 * T + 16 * g, have = a.features - f;
    const float xs = a.scale[p];
    float b[16];
    if (a.bias) load_row<float, 16>(a.bias + f, have, b);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const f32x4 ws = *(const f32x4*)(a.wscale + f + 4 * u);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[4 * u + r] = ((float)acc[u][r] * ws[r]) * xs;
            if (a.bias) v[4 * u + r] += b[4 * u + r];
        }
    }
    if (a.addend) {
        load16(a.addend, a.add_dtype, p * a.ldadd + f, have, b);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] += b[i];
    }
    if (a.relu) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // a NaN stays one
    }
}

template <int DT>
DEV void put(const LinearArgs& a, const i32x4 (&acc)[4], int T, int64_t p, int g) {
    const int f = 64 * T + 16 * g;
    if (f >= a.features) return;
    float v[16];
    finish_linear(a, acc, T, p, g, v);
    typedef typename Elem<DT>::T O;
    store_row<O, 16>((O*)a.out + p * a.ldout + f, a.features - f, v);
}

template <int DT>
DEV void put(const LinearArgs& a, const f32x4 (&acc)[4], int T, int64_t p, int g) {
    const int f = 64 * T + 16 * g;
    if (f >= a.features) return;
    unsigned bits = 0xffffu;
    if (a.mask) bits = *(const unsigned short*)(a.mask + p * (up64(a.features) / 8) + f / 8);
    float v[16];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[4 * u + r] = bits >> (4 * u + r) & 1 ? acc[u][r] : 0.f;
    typedef typename Elem<DT>::T O;
    store_row<O, 16>((O*)a.out + p * a.ldout + f, a.features - f, v);
}

// One wave: one group of 64 features x 16 P points, operands straight from global memory.
template <class Op, int DT, int P>
__global__ __launch_bounds__(256) void linear_direct_kernel(LinearArgs a) {
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int T = (int)(id % a.groups);
    const int64_t p0 = id / a.groups * (16 * P);
    if (p0 >= a.n) return;
    typename Op::Acc acc[P][4];
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[j][u] = Op::zero();
    int64_t row[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int64_t p = p0 + 16 * j + r;
        row[j] = p < a.n ? p : a.n - 1;  // a lane behind the last row repeats it and stores nothing
    }
    const char* w = a.frags + (size_t)T * a.steps * 4096 + lane * 16;
    for (int s = 0; s < a.steps; ++s, w += 4096) {
        typename Op::B b[P];
#pragma unroll
        for (int j = 0; j < P; ++j) b[j] = Op::load(a, row[j], s, g);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const i32x4 wf = *(const i32x4*)(w + u * 1024);
#pragma unroll
            for (int j = 0; j < P; ++j) acc[j][u] = Op::mma(wf, b[j], acc[j][u]);
        }
    }
#pragma unroll
    for (int j = 0; j < P; ++j)
        if (p0 + 16 * j + r < a.n) put<DT>(a, acc[j], T, row[j], g);
}

template <class Op, int DT>
static int launch(const LinearArgs& a, const char* what, hipStream_t st) {
    const int64_t waves = (a.n + 31) / 32 * a.groups;
    if ((waves + 3) / 4 >= (1LL << 24)) return NERF_FAIL(NERF_E_UNSUPPORTED, "%s: too many rows", what);
    linear_direct_kernel<Op, DT, 2><<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(a);
    return check_launch(what);
}

}  // namespace i8
}  // namespace nerf

using namespace nerf;
using namespace nerf::i8;

static int require_widths(const char* what, int64_t n, int k, int m) {
    NERF_REQUIRE(n >= 0 && k >= 1 && m >= 1 && k <= kMaxWidth && m <= kMaxWidth, "%s: bad size (%lld rows, %d x %d)", what, (long long)n, k, m);
    return 0;
}

NERF_API int nerf_linear_int8(const signed char* q, const float* scale, int64_t n, int k, const void* packed, int m,
                              const float* bias, const void* addend, int addend_dtype, int64_t ldadd, int relu, void* y,
                              int dtype, int64_t ldy, nerf_stream_t stream) {
    const char* what = "nerf_linear_int8";
    if (int rc = require_widths(what, n, k, m)) return rc;
    NERF_REQUIRE(dtype_ok(dtype) && (!addend || dtype_ok(addend_dtype)), "%s: unknown type", what);
    if (n == 0) return 0;
    NERF_REQUIRE(q && scale && packed && y, "%s: null pointer", what);
    NERF_REQUIRE(ldy >= m && (!addend || ldadd >= m), "%s: rows of %d elements overlap", what, m);
    NERF_REQUIRE((((uintptr_t)q | (uintptr_t)packed) & 15) == 0 && ((uintptr_t)y & (dtype_size(dtype) - 1)) == 0 &&
                     (((uintptr_t)scale | (uintptr_t)bias) & 3) == 0 && (!addend || ((uintptr_t)addend & (dtype_size(addend_dtype) - 1)) == 0),
                 "%s: misaligned pointer", what);
    const PackedLayout lay(k, m, false);
    LinearArgs a{};
    a.frags = (const char*)packed + lay.frags, a.groups = lay.mp / 64, a.steps = lay.kp / 64, a.n = n;
    a.q = q, a.scale = scale, a.features = m, a.wscale = (const float*)packed, a.bias = bias;
    a.addend = addend, a.add_dtype = addend_dtype, a.ldadd = ldadd, a.relu = relu, a.out = y, a.ldout = ldy;
    hipStream_t st = as_stream(stream);
    if (dtype == NERF_F32) return launch<Int8Op, NERF_F32>(a, what, st);
    if (dtype == NERF_F16) return launch<Int8Op, NERF_F16>(a, what, st);
    return launch<Int8Op, NERF_BF16>(a, what, st);
}

NERF_API int nerf_linear_int8_grad_input(const void* dz, int dtype, int64_t n, int m, int64_t lddz, const void* packed,
                                         int k, const unsigned char* mask, void* dx, int64_t lddx, nerf_stream_t stream) {
    const char* what = "nerf_linear_int8_grad_input";
    if (int rc = require_widths(what, n, k, m)) return rc;
    NERF_REQUIRE(dtype_ok(dtype), "%s: unknown type %d", what, dtype);
    if (n == 0) return 0;
    NERF_REQUIRE(dz && packed && dx, "%s: null pointer", what);
    NERF_REQUIRE(lddz >= m && lddx >= k, "%s: rows overlap", what);
    NERF_REQUIRE(((uintptr_t)packed & 15) == 0 && (((uintptr_t)dz | (uintptr_t)dx) & (dtype_size(dtype) - 1)) == 0 &&
                     ((uintptr_t)mask & 1) == 0,
                 "%s: misaligned pointer", what);
    const PackedLayout lay(k, m, true);
    LinearArgs a{};
    a.frags = (const char*)packed + lay.frags_t, a.groups = lay.kp / 64, a.steps = lay.mp / 32, a.n = n;
    a.dz = dz, a.lddz = lddz, a.width = m, a.features = k, a.mask = mask, a.out = dx, a.ldout = lddx;
    hipStream_t st = as_stream(stream);
    if (dtype == NERF_F32) return launch<Bf16Op<NERF_F32>, NERF_F32>(a, what, st);
    if (dtype == NERF_F16) return launch<Bf16Op<NERF_F16>, NERF_F16>(a, what, st);
    return launch<Bf16Op<NERF_BF16>, NERF_BF16>(a, what, st);
}
