// Products of rows with packed weights, shared by int8_linear.hip (8-bit integers, int32 sums) and
// int8_grad_input.hip (bf16 terms, fp32 sums).  Formats: int8_common.h.
//
// Both are D[feature][point] = sum over the contraction of A[feature][c] B[c][point] with 16 x 16 tiles: a
// lane's B fragment is 16 integers (8 bf16) that lie next to each other in its point's row.  Which
// features a tile has is a matter of the rows its A fragment is read with (frag_source): the four tiles of
// a group of 64 features leave a lane (point = lane & 15, g = lane >> 4) pieces of 16 bytes of the
// output, 4, 8 or 16 neighbouring features, and the four lanes of a point pieces that are neighbours, so
// that every store covers 64-byte runs.
#pragma once
#include "int8_common.h"
#include "mlp_common.h"

namespace nerf {
namespace i8 {

struct LinearArgs {
    const char* frags;     // this product's fragments
    int groups, steps;     // groups of 64 features, steps of 64 integers (32 bf16) of the rows
    int frag_steps;        // ... of the fragments (bf16: one more where the rows end in the first half of 64)
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
    const void* addend;    // [n][ldadd] of the type the kernel is instantiated for
    int64_t ldadd;
    int relu;
    const unsigned char* mask;
    void* out;
    int64_t ldout;
    // output in 8 bits (TO_INT8): out = integers, and
    float* out_scale;
    unsigned char* out_mask;
    unsigned* tops;        // of rows beyond one workgroup: [n][feature blocks] largest magnitudes
    int pass;              // ... 1: they are formed, 2: they are read; 0: a row is one workgroup's
};

// What a product is stored as: a type (NERF_F32, ...) or 8-bit rows: TO_INT8, + 1 behind a ReLU, + 2 with
// scales that are powers of two.
constexpr int TO_INT8 = 4;
// Type of an addend: NERF_F32 or NERF_BF16 (fp16 is exact in fp32), or none.
constexpr int NO_ADD = -1;

// ---- the two products -----------------------------------------------------------------------------
// Raw: what a lane loads of a point's row for one step; B: the operands made of it.
struct Int8Op {
    typedef i32x4 Acc;
    typedef i32x4 Raw;
    static constexpr bool kInt8 = true;
    static DEV Raw fetch(const LinearArgs& a, int64_t p, int s, int g) {
        return *(const i32x4*)(a.q + (p * a.steps + s) * 64 + 16 * g);
    }
    struct B {
        i32x4 v;
        DEV B(const Raw& r) : v(r) {}
    };
    static DEV Raw raw_of(i32x4 w) { return w; }
    static DEV Acc mma(i32x4 w, const B& b, Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, b.v, c, 0, 0, 0); }
};

// EVEN: the rows of dz end with a step (32 columns), so that no piece of one needs the care of a ragged end.
template <int DT, bool EVEN>
struct Bf16Op {
    typedef f32x4 Acc;
    typedef typename Elem<DT>::T T;
    typedef Raw8<T> Raw;
    static constexpr bool kInt8 = false;
    static constexpr int N = Terms<DT>::N;
    static DEV Raw fetch(const LinearArgs& a, int64_t p, int s, int g) {
        return load8<T>((const T*)a.dz + p * a.lddz, 32 * s + 8 * g, a.width, EVEN || 32 * s + 32 <= a.width);
    }
    static DEV Raw raw_of(i32x4 w) {  // 16-bit types
        Raw r;
        r.w[0] = w;
        return r;
    }
    struct B {
        bf16x8 v[N];
        DEV B(const Raw& r) {
            if constexpr (DT == NERF_BF16) {
                v[0] = __builtin_bit_cast(bf16x8, r.w[0]);
            } else {
                float f[8];
                to_float(r, f);
                split_bf16<N>(f, v);
            }
        }
    };
    static DEV Acc mma(i32x4 w, const B& b, Acc c) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), b.v[i], c, 0, 0, 0);
        return c;
    }
};

// ---- which features a lane has -------------------------------------------------------------------------
template <int OUT> constexpr int kPiece = OUT == NERF_F32 ? 4 : OUT < TO_INT8 ? 8 : 16;

// Feature, inside its group of 64, of value i of a lane (accumulator i >> 2, register i & 3).
template <int OUT>
DEV int feature_of(int i, int g) {
    return (i / kPiece<OUT>) * (4 * kPiece<OUT>) + g * kPiece<OUT> + i % kPiece<OUT>;
}
// Where, in the four stored fragments of a group and step, a lane finds its row of A for tile u.
template <int OUT>
DEV int frag_source(int u, int lane) {
    const int f = feature_of<OUT>(4 * u + (lane & 3), (lane >> 2) & 3);
    return ((f >> 2) & 3) * 1024 + (4 * (f >> 4) + (f & 3) + (lane & 48)) * 16;
}

// ---- what becomes of the sums of a lane ------------------------------------------------------------------
// N neighbouring elements of a row added to v; `whole` (the same in every lane): all of them exist.
template <class A, int N>
DEV void add_piece(const A* p, int have, bool whole, float* v) {
    if (whole) {
        constexpr int W = N * sizeof(A) / 4;
        int w[W];
        if constexpr (W == 2) {
            typedef int i32x2 __attribute__((ext_vector_type(2)));
            const i32x2 q = *(const i32x2u*)p;
            w[0] = q[0], w[1] = q[1];
        } else {
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                const i32x4 q = *(const i32x4u*)((const char*)p + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = q[j];
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (sizeof(A) == 4) v[i] += __builtin_bit_cast(float, w[i]);
            else v[i] += __builtin_bit_cast(float, (i & 1) ? w[i >> 1] & (int)0xffff0000 : w[i >> 1] << 16);  // bf16
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < have) v[i] += (float)p[i];
    }
}

// 16 bytes of a row, as far as its elements exist: a piece that passes the end leaves as runs of 4, 2 and 1.
template <class T, int N>
DEV void store_piece(T* dst, int have, bool whole, const float* v) {
    int w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (N == 4) {
            w[i] = __builtin_bit_cast(int, v[i]);
        } else {
            typedef T pair __attribute__((ext_vector_type(2)));
            const pair t = {(T)v[2 * i], (T)v[2 * i + 1]};
            w[i] = __builtin_bit_cast(int, t);
        }
    }
    if (whole || have >= N) {
        if constexpr (N == 8) {
            // a row that starts between two words: the words inside the piece as such, half of one at each end
            // (a vector store is slow there only)
            if ((uintptr_t)dst & 2) {
                typedef int i32x3u __attribute__((ext_vector_type(3), aligned(4)));
                char* d = (char*)dst;
                *(unsigned short*)d = (unsigned short)w[0];
                *(i32x3u*)(d + 2) = i32x3u{(int)__builtin_amdgcn_alignbit(w[1], w[0], 16), (int)__builtin_amdgcn_alignbit(w[2], w[1], 16),
                                           (int)__builtin_amdgcn_alignbit(w[3], w[2], 16)};
                *(unsigned short*)(d + 14) = (unsigned short)((unsigned)w[3] >> 16);
                return;
            }
        }
        *(i32x4u*)dst = i32x4{w[0], w[1], w[2], w[3]};
        return;
    }
    if (have <= 0) return;
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    char* d = (char*)dst;
    const int words = have * (int)sizeof(T) / 4;
    if (words & 2) {
        *(i32x2u*)d = i32x2{w[0], w[1]};
        d += 8, w[0] = w[2], w[1] = w[3];
    }
    if (words & 1) {
        *(i32u*)d = w[0];
        d += 4, w[0] = w[1];
    }
    if constexpr (N == 8) {
        if (have & 1) *(unsigned short*)d = (unsigned short)w[0];
    }
}

// y = relu((sum x channel scale) x row scale + bias + addend): the sum rounded to fp32, its product with
// the channel scale rounded, then one rounding for row scale and bias and one for the addend.  ws, b: the
// channels' scales and biases of the group of 64 from f0 (0 and 0 behind the last channel).
template <int OUT, int ADD>
DEV void finish_linear(const LinearArgs& a, const i32x4 (&acc)[4], const float* ws, const float* b, float xs, int f0, int g,
                       int64_t p, bool whole, bool relu, float (&v)[16]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int f = feature_of<OUT>(4 * u, g);
        const f32x4 w4 = *(const f32x4*)(ws + f), b4 = *(const f32x4*)(b + f);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[4 * u + r] = __builtin_fmaf((float)acc[u][r] * w4[r], xs, b4[r]);
    }
    if constexpr (ADD != NO_ADD) {
        typedef typename Elem<ADD>::T A;
        const A* row = (const A*)a.addend + p * a.ldadd;
#pragma unroll
        for (int i = 0; i < 16; i += kPiece<OUT>) {
            const int f = f0 + feature_of<OUT>(i, g);
            add_piece<A, kPiece<OUT>>(row + f, a.features - f, whole, v + i);
        }
    }
    if (relu) {  // (v_maximum3_f32: a NaN of either sign stays one)
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __builtin_elementwise_maximum(v[i], 0.f);
    }
}

// One bit per value: v > 0.  Behind a ReLU (and without a NaN) that is a bit pattern other than zero, the
// sign of its negative: a subtraction and a funnel shift a value (a comparison's result takes two wait
// states to be read, and a selection to become a bit).
template <bool RELU>
DEV unsigned positive_bits(const float (&v)[16], bool has_nan) {
    unsigned bits = 0u;
    if (RELU && __builtin_expect(!has_nan, 1)) {
#pragma unroll
        for (int i = 15; i >= 0; --i) bits = __builtin_amdgcn_alignbit(bits, 0u - __builtin_bit_cast(unsigned, v[i]), 31);
    } else {
        if constexpr (RELU) asm volatile("");  // a branch that is hardly ever taken, not a selection between both
#pragma unroll
        for (int i = 0; i < 16; ++i) bits |= v[i] > 0.f ? 1u << i : 0u;
    }
    return bits;
}

// 16 values in bytes.  POW2: the product is exact, so the addition may take it in unrounded.
template <bool POW2>
DEV uint4 round16(const float (&v)[16], float inv) {
    unsigned o[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        float t[4];
#pragma unroll
        for (int b = 0; b < 4; ++b)
            t[b] = POW2 ? __builtin_fmaf(v[4 * w + b], inv, kRoundAt) : v[4 * w + b] * inv + kRoundAt;
        o[w] = low_bytes(t);
    }
    return inv == 0.f ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(o[0], o[1], o[2], o[3]);
}

template <int OUT>
DEV void put(const LinearArgs& a, int64_t p, int f0, int g, bool whole, const float (&v)[16]) {
    typedef typename Elem<OUT>::T O;
    O* row = (O*)a.out + p * a.ldout;
#pragma unroll
    for (int i = 0; i < 16; i += kPiece<OUT>) {
        const int f = f0 + feature_of<OUT>(i, g);
        store_piece<O, kPiece<OUT>>(row + f, a.features - f, whole, v + i);
    }
}

// The 64 bits of a group of features, moved so that a lane's own are at places that do not depend on it.
template <int OUT>
DEV uint2 own_bits(uint2 m, int g) {
    return make_uint2(m.x >> (g * kPiece<OUT>), m.y >> (g * kPiece<OUT>));
}

template <int OUT>
DEV void put_grad(const LinearArgs& a, const f32x4 (&acc)[4], int f0, int g, int64_t p, bool whole, uint2 own) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int at = (i / kPiece<OUT>) * (4 * kPiece<OUT>) + i % kPiece<OUT>;  // of 64, but for the lane's shift
        const float x = acc[i >> 2][i & 3];
        const int keep = __builtin_amdgcn_sbfe((int)(at < 32 ? own.x : own.y), at & 31, 1);  // all ones or none
        v[i] = __builtin_bit_cast(float, __builtin_bit_cast(int, x) & keep);
    }
    put<OUT>(a, p, f0, g, whole, v);
}

// Channel scales and biases of `count` features from f0 into LDS, zeros behind the last.
DEV void stage_channels(const LinearArgs& a, float* ws, float* b, int f0, int count) {
    for (int i = threadIdx.x; i < count; i += blockDim.x) {
        const int f = f0 + i;
        ws[i] = f < a.features ? a.wscale[f] : 0.f;
        b[i] = (a.bias && f < a.features) ? a.bias[f] : 0.f;
    }
}

// ---- kernels --------------------------------------------------------------------------------------------

// Few rows: one wave per group of 64 features x 32 points, operands straight from global memory.
template <class Op, int OUT, int ADD>
__global__ __launch_bounds__(256) void linear_direct_kernel(LinearArgs a) {
    constexpr int P = 2;
    __shared__ __attribute__((aligned(16))) float ch[4][2][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int64_t id = (int64_t)blockIdx.x * 4 + wave;
    const int T = (int)(id % a.groups);
    const int64_t p0 = id / a.groups * (16 * P);
    if (p0 >= a.n) return;
    typename Op::Acc acc[P][4];
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[j][u] = typename Op::Acc{};
    int64_t row[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int64_t p = p0 + 16 * j + r;
        row[j] = p < a.n ? p : a.n - 1;  // a lane behind the last row repeats it and stores nothing
    }
    const char* w = a.frags + (size_t)T * a.frag_steps * 4096;
    int at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) at[u] = frag_source<OUT>(u, lane);
    for (int s = 0; s < a.steps; ++s, w += 4096) {
        typename Op::Raw raw[P];
#pragma unroll
        for (int j = 0; j < P; ++j) raw[j] = Op::fetch(a, row[j], s, g);
        i32x4 wf[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) wf[u] = *(const i32x4*)(w + at[u]);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const typename Op::B b(raw[j]);
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[j][u] = Op::mma(wf[u], b, acc[j][u]);
        }
    }
    const bool whole = 64 * T + 64 <= a.features;
    if constexpr (Op::kInt8) {
        // this wave's 64 channels, through its own piece of LDS (one wave: in order, no barrier)
        const int c = 64 * T + lane;
        ch[wave][0][lane] = c < a.features ? a.wscale[c] : 0.f;
        ch[wave][1][lane] = (a.bias && c < a.features) ? a.bias[c] : 0.f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < P; ++j) {
            float v[16];
            finish_linear<OUT, ADD>(a, acc[j], ch[wave][0], ch[wave][1], a.scale[row[j]], 64 * T, g, row[j], whole, a.relu != 0, v);
            if (p0 + 16 * j + r < a.n) put<OUT>(a, row[j], 64 * T, g, whole, v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint2 m = a.mask ? *(const uint2*)(a.mask + row[j] * (a.groups * 8) + 8 * T) : make_uint2(~0u, ~0u);
            if (p0 + 16 * j + r < a.n) put_grad<OUT>(a, acc[j], 64 * T, g, row[j], whole, own_bits<OUT>(m, g));
        }
    }
}

// Many rows, weights that fit LDS: a workgroup per CU copies the fragments of up to NT groups of
// features into LDS once and its eight waves then stream tiles of 16 P points past them.  A wave holds
// the sums of all NT groups of a tile (16 NT P registers), so a row is read once, and its work is a run of
// units: CH steps of a tile's rows.  While one unit is worked on, the next one's rows (of this tile or the
// next) are on their way into the other half of the registers, so that loads are in flight all the
// time; with bf16 rows, tiles of 32 points, which halve the reads of LDS, leave no room for that (786432 x
// 256 x 256, input gradient: 249 us against 172; 8-bit rows are small enough for two tiles of 16 and both
// halves).  A fetch is the same loads on every path (a step behind the last repeats it, a tile behind the
// last repeats the one at hand): a wait for older loads counts the younger ones.
// Bound by memory up to a few hundred inputs and outputs: 786432 x 256 x 256 bf16 input gradient 172 us
// (4.8 TB/s), 262144 x 319 x 256 -> bf16 46 us (4.7 TB/s); with 8-bit output by vector instructions
// (786432 x 256 x 256: 116 us, 3.6 TB/s, about 8 of them a value).
constexpr int kResidentThreads = 512;
template <int NT>
constexpr int channel_bytes() { return 2 * NT * 64 * 4; }

template <class Op, int OUT, int NT, int CH, int P, int ADD>
__global__ __launch_bounds__(kResidentThreads) void linear_resident_kernel(LinearArgs a, int64_t tiles) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* const ws = (float*)lds;
    float* const bs = ws + NT * 64;
    char* const wl = lds + channel_bytes<NT>();
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int T0 = blockIdx.y * NT;

    // what the work on a tile's sums reads of its rows: requested with them, not when it is needed (that
    // wait would also be one for the next unit's rows)
    struct Side {
        float xs;
        uint2 bits[NT];
    };
    typename Op::Raw raw[2][CH][P];
    Side side[2][P];  // of the tile being worked on, of the one being fetched
    typename Op::Acc acc[P][NT][4];
    auto row_of = [&](int64_t tile, int j) {
        const int64_t p = tile * (16 * P) + 16 * j + r;
        return p < a.n ? p : a.n - 1;  // a lane behind the last row repeats it and stores nothing
    };
    // bits of the mask: without one, any bytes, all set afterwards
    const unsigned char* const mask = a.mask ? a.mask : (const unsigned char*)a.frags;
    const int64_t mask_ld = a.mask ? a.groups * 8 : 0;
    const unsigned no_mask = a.mask ? 0u : ~0u;
    auto fetch = [&](int64_t tile, int s0, typename Op::Raw (&to)[CH][P]) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int64_t p = row_of(tile, j);
            if constexpr (Op::kInt8) {
                side[1][j].xs = a.scale[p];
            } else {
#pragma unroll
                for (int T = 0; T < NT; ++T) {
                    const int t = T0 + T < a.groups ? T0 + T : a.groups - 1;
                    const uint2 m = *(const uint2*)(mask + p * mask_ld + 8 * t);
                    side[1][j].bits[T] = make_uint2(m.x | no_mask, m.y | no_mask);
                }
            }
#pragma unroll
            for (int i = 0; i < CH; ++i) to[i][j] = Op::fetch(a, p, s0 + i < a.steps ? s0 + i : a.steps - 1, g);
        }
    };
    auto multiply = [&](int s0, const typename Op::Raw (&from)[CH][P]) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (i == 0 || s0 + i < a.steps) {  // a unit has at least one step
                const char* w = wl + (s0 + i) * (NT * 4096) + lane * 16;
                if constexpr (P == 1) {
                    const typename Op::B b(from[i][0]);
#pragma unroll
                    for (int T = 0; T < NT; ++T)
#pragma unroll
                        for (int u = 0; u < 4; ++u) acc[0][T][u] = Op::mma(*(const i32x4*)(w + (T * 4 + u) * 1024), b, acc[0][T][u]);
                } else {
                    const typename Op::B b0(from[i][0]), b1(from[i][1]);
#pragma unroll
                    for (int T = 0; T < NT; ++T)
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const i32x4 wf = *(const i32x4*)(w + (T * 4 + u) * 1024);
                            acc[0][T][u] = Op::mma(wf, b0, acc[0][T][u]);
                            acc[1][T][u] = Op::mma(wf, b1, acc[1][T][u]);
                        }
                }
            }
        }
    };
    auto finish = [&](int64_t tile) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int64_t p = row_of(tile, j);
            const bool live = tile * (16 * P) + 16 * j + r < a.n;
            const Side& now = side[0][j];
            if constexpr (!Op::kInt8) {
                if (live) {
#pragma unroll
                    for (int T = 0; T < NT; ++T) {
                        if (T0 + T < a.groups)
                            put_grad<OUT>(a, acc[j][T], 64 * (T0 + T), g, p, 64 * (T0 + T) + 64 <= a.features, own_bits<OUT>(now.bits[T], g));
                    }
                }
            } else if constexpr (OUT < TO_INT8) {
#pragma unroll
                for (int T = 0; T < NT; ++T) {
                    const bool whole = 64 * (T0 + T) + 64 <= a.features;
                    if (T0 + T < a.groups && live) {
                        float v[16];
                        finish_linear<OUT, ADD>(a, acc[j][T], ws + 64 * T, bs + 64 * T, now.xs, 64 * (T0 + T), g, p, whole, a.relu != 0, v);
                        put<OUT>(a, p, 64 * (T0 + T), g, whole, v);
                    }
                    __builtin_amdgcn_sched_barrier(0);  // in turn: 16 sums become 16 values in the same registers
                }
            } else {
                // the whole row is here (16 features per group in each of 4 lanes): its scale, then its integers
                constexpr bool RELU = (OUT & 1) != 0, POW2 = (OUT & 2) != 0;
                float v[NT][16];
                unsigned top = 0u;
#pragma unroll
                for (int T = 0; T < NT; ++T) {
                    if (T < a.groups) {  // (an addend's rows are whole groups here)
                        finish_linear<OUT, ADD>(a, acc[j][T], ws + 64 * T, bs + 64 * T, now.xs, 64 * T, g, p, true, RELU, v[T]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[T][i] = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const unsigned m = RELU ? __builtin_bit_cast(unsigned, v[T][i]) : magnitude(v[T][i]);
                        top = top > m ? top : m;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int off = 16; off < 64; off *= 2) {
                    const unsigned o = (unsigned)__shfl_xor((int)top, off);
                    top = top > o ? top : o;
                }
                const Scale sc = scale_of(top, POW2);
                const bool has_nan = __any(top > 0x7f800000u);
                const int fp = a.groups * 64;  // width of a row of the output
                if (live && g == 0) a.out_scale[p] = sc.scale;
#pragma unroll
                for (int T = 0; T < NT; ++T) {
                    if (T < a.groups) {
                        const uint4 o = round16<POW2>(v[T], sc.inv);
                        if (live) *(uint4*)((signed char*)a.out + p * fp + 64 * T + 16 * g) = o;
                        if (a.out_mask) {
                            const unsigned bits = positive_bits<RELU>(v[T], has_nan);
                            if (live) *(unsigned short*)(a.out_mask + p * (fp / 8) + 8 * T + 2 * g) = (unsigned short)bits;
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };

    // The first rows are requested, then the fragments are copied, [group][step] -> LDS [step][group], without
    // passing registers (a group behind the last repeats it and is not stored), all before the first wait.
    const int64_t stride = (int64_t)gridDim.x * (kResidentThreads / 64);
    int64_t tile = (int64_t)blockIdx.x * (kResidentThreads / 64) + wave;
    int s0 = 0;
    fetch(tile < tiles ? tile : tiles - 1, 0, raw[0]);
    const int lane_source = frag_source<OUT>(wave & 3, lane);  // this wave copies tile wave & 3 of every group and step
    for (int i = wave; i < NT * a.steps * 4; i += kResidentThreads / 64) {
        const int s = i / (NT * 4), T = (i >> 2) % NT, t = T0 + T < a.groups ? T0 + T : a.groups - 1;
        glds16_untracked(a.frags + ((size_t)t * a.frag_steps + s) * 4096 + lane_source, wl + i * 1024);
    }
    if constexpr (Op::kInt8) stage_channels(a, ws, bs, 64 * T0, NT * 64);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    while (tile < tiles) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (tile >= tiles) break;
            const bool last = s0 + CH >= a.steps;
            const int64_t tile1 = last ? tile + stride : tile;
            const int s1 = last ? 0 : s0 + CH;
            if (s0 == 0) {
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    side[0][j] = side[1][j];
#pragma unroll
                    for (int T = 0; T < NT; ++T)
#pragma unroll
                        for (int u = 0; u < 4; ++u) acc[j][T][u] = typename Op::Acc{};
                }
            }
            fetch(tile1 < tiles ? tile1 : tile, s1, raw[h ^ 1]);
            multiply(s0, raw[h]);
            if (last) finish(tile);
            tile = tile1, s0 = s1;
        }
    }
}

// Weights that do not fit LDS: a workgroup forms a tile of 128 FW features x 512 / FW points, a wave 128 x 64
// of it (128 registers of sums), FW waves side by side along the features.  The contraction goes through a
// ring of stages of one step (8 FW fragments of weights, 32 / FW of rows), copied from global memory to LDS
// without passing registers, all but one stage ahead; per stage a wave reads 12 fragments for 32
// products, so the matrix unit and not LDS sets the pace.  Rows must be 16-byte aligned and end with a
// step.  Workgroups 8 apart run on the same die: they take the feature blocks of one block of rows in turn,
// which the die's L2 then holds.  Bound by the matrix unit: 32768 x 2048 x 2048 144 us, 1.9 P op/s (weights
// and rows straight from memory: 253 us).
// FW 2: tiles of 256 x 256 and four stages of 32 KiB.  FW 4: 512 x 128 and three of 40 KiB, for 8-bit output of
// 257 to 512 features, whose scale takes the whole row: the waves' maxima meet in LDS.  Longer rows with 8-bit
// output are formed twice, first for their blocks' maxima, then for their integers.
constexpr int kStreamThreads = 512;
template <int FW> constexpr int kStreamStages = FW == 2 ? 4 : 3;
template <int FW> constexpr int kStreamStage = (8 * FW + 32 / FW) * 1024;
template <int FW> constexpr int kStreamPoints = 512 / FW;
template <int FW> constexpr int kStreamLds = 2 * 128 * FW * 4 + FW * kStreamPoints<FW> * 4 + kStreamStages<FW> * kStreamStage<FW>;

template <class Op, int OUT, int ADD, int FW>
__global__ __launch_bounds__(kStreamThreads) void linear_streamed_kernel(LinearArgs a, int fblocks, int64_t pblocks) {
    static_assert(FW == 2 || FW == 4, "shapes");
    constexpr int kFeatures = 128 * FW, kPoints = kStreamPoints<FW>, S = kStreamStages<FW>;
    constexpr int C = (8 * FW + 32 / FW) / 8;  // copies of a wave for a stage
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* const ws = (float*)lds;
    float* const bs = ws + kFeatures;
    unsigned* const tops = (unsigned*)(bs + kFeatures);  // [FW][kPoints]
    char* const ring = (char*)(tops + FW * kPoints);
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fb = (int)(blockIdx.x / 8 % fblocks);
    const int64_t pb = (int64_t)(blockIdx.x / 8 / fblocks) * 8 + (blockIdx.x & 7);
    if (pb >= pblocks) return;  // the whole workgroup
    const int T0 = 2 * FW * fb;

    // this wave's copies of a stage: the four fragments of a group of features (waves below 2 FW), fragments of
    // rows (FW 2: four by each of the other waves; FW 4: one by every wave)
    const char* src[C];
    const auto row = [&](int frag) {
        int64_t p = pb * kPoints + frag * 16 + r;
        if (p >= a.n) p = a.n - 1;
        if constexpr (Op::kInt8) return (const char*)a.q + p * a.steps * 64 + 16 * g;
        else return (const char*)a.dz + p * a.lddz * 2 + 16 * g;
    };
    const bool has_weights = FW == 4 || wave < 4;
    const int step = has_weights ? 4096 : 64;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        if (i < 4 && has_weights) {
            const int T = T0 + wave < a.groups ? T0 + wave : a.groups - 1;  // a group behind the last is not stored
            src[i] = a.frags + (size_t)T * a.frag_steps * 4096 + frag_source<OUT>(i & 3, lane);
        } else {
            src[i] = row(FW == 4 ? wave : (wave - 4) * 4 + i);
        }
    }
    auto issue = [&](int s) {
        char* st = ring + (s % S) * kStreamStage<FW>;
#pragma unroll
        for (int i = 0; i < C; ++i)
            glds16_untracked(src[i] + (int64_t)s * (i < 4 ? step : 64), st + (i < 4 ? wave * 4 + i : 8 * FW + wave) * 1024);
    };

    if constexpr (Op::kInt8) {
        stage_channels(a, ws, bs, 64 * T0, kFeatures);  // read behind the barriers of the loop
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing but the copies is counted from here on
    }
    const int wf = wave % FW, wp = wave / FW;
    typename Op::Acc acc[4][2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[j][t][u] = typename Op::Acc{};
#pragma unroll
    for (int s = 0; s < S - 1; ++s)
        if (s < a.steps) issue(s);
    for (int s = 0; s < a.steps; ++s) {
        // this wave's copies of stage s have arrived (the younger stages may be on their way), then everyone's
        const int younger = a.steps - 1 - s;
        if (younger >= S - 2) wait_vmcnt_n(C * (S - 2));
        else if (S > 3 && younger == 1) wait_vmcnt_n(C);
        else wait_vmcnt_n(0);
        // (lgkmcnt: this wave's reads of the stage that is overwritten next have arrived)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + S - 1 < a.steps) issue(s + S - 1);
        const char* st = ring + (s % S) * kStreamStage<FW> + lane * 16;
        const char* wl = st + wf * 8 * 1024;
        const char* xl = st + 8 * FW * 1024 + wp * 4 * 1024;
        const auto rows = [&](int j) { return typename Op::B(Op::raw_of(*(const i32x4*)(xl + j * 1024))); };
        const typename Op::B b[4] = {rows(0), rows(1), rows(2), rows(3)};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const i32x4 wfr = *(const i32x4*)(wl + (4 * t + u) * 1024);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j][t][u] = Op::mma(wfr, b[j], acc[j][t][u]);
            }
    }
    const int64_t p0 = pb * kPoints + wp * 64 + r;
    if constexpr (OUT < TO_INT8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool live = p0 + 16 * j < a.n;
            const int64_t p = live ? p0 + 16 * j : a.n - 1;
            float xs = 0.f;
            if constexpr (Op::kInt8) xs = a.scale[p];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int T = 2 * wf + t;
                const bool whole = 64 * (T0 + T) + 64 <= a.features;
                if (T0 + T < a.groups) {
                    if constexpr (Op::kInt8) {
                        float v[16];
                        finish_linear<OUT, ADD>(a, acc[j][t], ws + 64 * T, bs + 64 * T, xs, 64 * (T0 + T), g, p, whole, a.relu != 0, v);
                        if (live) put<OUT>(a, p, 64 * (T0 + T), g, whole, v);
                    } else if (live) {
                        const uint2 m = a.mask ? *(const uint2*)(a.mask + p * (a.groups * 8) + 8 * (T0 + T)) : make_uint2(~0u, ~0u);
                        put_grad<OUT>(a, acc[j][t], 64 * (T0 + T), g, p, whole, own_bits<OUT>(m, g));
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    } else {
        // the largest of a point's features in this wave, in all FW that share it, and in all workgroups
        constexpr bool RELU = (OUT & 1) != 0, POW2 = (OUT & 2) != 0;
        float v[4][2][16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t p = p0 + 16 * j < a.n ? p0 + 16 * j : a.n - 1;
            const float xs = a.scale[p];
            unsigned top = 0u;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int T = 2 * wf + t;
                if (T0 + T < a.groups) {  // (an addend's rows are whole groups here)
                    finish_linear<OUT, ADD>(a, acc[j][t], ws + 64 * T, bs + 64 * T, xs, 64 * (T0 + T), g, p, true, RELU, v[j][t]);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[j][t][i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const unsigned m = RELU ? __builtin_bit_cast(unsigned, v[j][t][i]) : magnitude(v[j][t][i]);
                    top = top > m ? top : m;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int off = 16; off < 64; off *= 2) {
                const unsigned o = (unsigned)__shfl_xor((int)top, off);
                top = top > o ? top : o;
            }
            if (g == 0 && a.pass != 2) tops[wf * kPoints + wp * 64 + 16 * j + r] = top;
        }
        if (a.pass == 2) {
            const int64_t p = pb * kPoints + threadIdx.x % kPoints;
            unsigned top = 0u;
            if (p < a.n)
                for (int i = threadIdx.x / kPoints; i < fblocks; i += FW) top = top > a.tops[p * fblocks + i] ? top : a.tops[p * fblocks + i];
            tops[threadIdx.x] = top;  // [FW][kPoints]: kStreamThreads
        }
        __syncthreads();
        if (a.pass == 1) {
            const int64_t p = pb * kPoints + threadIdx.x;
            if (threadIdx.x < kPoints && p < a.n) {
                unsigned top = 0u;
                for (int w = 0; w < FW; ++w) top = top > tops[w * kPoints + threadIdx.x] ? top : tops[w * kPoints + threadIdx.x];
                a.tops[p * fblocks + fb] = top;
            }
            return;
        }
        const int fp = a.groups * 64;  // width of a row of the output
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t p = p0 + 16 * j;
            const bool live = p < a.n;
            unsigned top = 0u;
#pragma unroll
            for (int w = 0; w < FW; ++w) {
                const unsigned o = tops[w * kPoints + wp * 64 + 16 * j + r];
                top = top > o ? top : o;
            }
            const Scale sc = scale_of(top, POW2);
            const bool has_nan = __any(top > 0x7f800000u);
            if (live && g == 0 && wf == 0 && fb == 0) a.out_scale[p] = sc.scale;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int T = 2 * wf + t;
                if (T0 + T < a.groups) {
                    const uint4 o = round16<POW2>(v[j][t], sc.inv);
                    if (live) *(uint4*)((signed char*)a.out + p * fp + 64 * (T0 + T) + 16 * g) = o;
                    if (a.out_mask) {
                        const unsigned bits = positive_bits<RELU>(v[j][t], has_nan);
                        if (live) *(unsigned short*)(a.out_mask + p * (fp / 8) + 8 * (T0 + T) + 2 * g) = (unsigned short)bits;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
}

constexpr int kLdsBytes = 160 * 1024;

template <class Op, int OUT, int NT, int CH, int P, int ADD>
int launch_resident(const LinearArgs& a, const char* what, hipStream_t st) {
    const size_t lds = channel_bytes<NT>() + (size_t)NT * a.steps * 4096;
    auto kernel = linear_resident_kernel<Op, OUT, NT, CH, P, ADD>;
    // (the limit is an attribute of the function on every device; asking again costs nothing)
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
    if (e != hipSuccess) return NERF_FAIL((int)e, "%s: %s", what, hipGetErrorString(e));
    int cus = device_cu_count();
    if (cus <= 0) cus = 256;
    const int64_t tiles = (a.n + 16 * P - 1) / (16 * P);
    const int fblocks = (a.groups + NT - 1) / NT;
    int64_t blocks = (tiles + kResidentThreads / 64 - 1) / (kResidentThreads / 64);
    const int64_t most = cus / fblocks > 0 ? cus / fblocks : 1;
    if (blocks > most) blocks = most;
    kernel<<<dim3((unsigned)blocks, (unsigned)fblocks), kResidentThreads, lds, st>>>(a, tiles);
    return check_launch(what);
}

template <class Op, int OUT, int ADD, int FW>
int launch_streamed(const LinearArgs& a, const char* what, hipStream_t st) {
    static_assert(kStreamLds<FW> <= kLdsBytes, "does not fit");
    auto kernel = linear_streamed_kernel<Op, OUT, ADD, FW>;
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
    if (e != hipSuccess) return NERF_FAIL((int)e, "%s: %s", what, hipGetErrorString(e));
    const int fblocks = (a.groups + 2 * FW - 1) / (2 * FW);
    static_assert(FW * kStreamPoints<FW> == kStreamThreads, "a thread per maximum");
    const int64_t pblocks = (a.n + kStreamPoints<FW> - 1) / kStreamPoints<FW>, grid = (pblocks + 7) / 8 * 8 * fblocks;
    if (grid >= (1LL << 23)) return NERF_FAIL(NERF_E_UNSUPPORTED, "%s: too many rows", what);  // fewer than 2^32 work items
    kernel<<<(unsigned)grid, kStreamThreads, kStreamLds<FW>, st>>>(a, fblocks, pblocks);
    return check_launch(what);
}

template <class Op, int DT, int ADD>
int launch_direct(const LinearArgs& a, const char* what, hipStream_t st) {
    const int64_t waves = (a.n + 31) / 32 * a.groups;
    if ((waves + 3) / 4 >= (1LL << 24)) return NERF_FAIL(NERF_E_UNSUPPORTED, "%s: too many rows", what);
    linear_direct_kernel<Op, DT, ADD><<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(a);
    return check_launch(what);
}

inline int require_widths(const char* what, int64_t n, int k, int m) {
    NERF_REQUIRE(n >= 0 && k >= 1 && m >= 1 && k <= kMaxWidth && m <= kMaxWidth, "%s: bad size (%lld rows, %d x %d)", what, (long long)n, k, m);
    return 0;
}

// Few enough rows for the direct kernel, whose time goes with its work (each wave reads its rows' and features'
// operands again) where the others begin with a copy of weights per CU or a tile of 256 points.  us, direct and
// resident: 256 x 256 to bf16, 4096 rows 4.5, 10.3, 16384 rows 6.9, 11.1, 32768 rows 11.1, 11.8, 65536 rows 18.7,
// 13.7; 63 x 256 at 32768 and 65536 rows 7.3, 9.0 and 11.6, 10.7; bf16 gradient of 256 x 256 at 16384 rows 9.4, 10.0, at
// 32768 16.9, 11.0.  Direct and streamed: 512 x 512, 8192 rows 9.3, 14.2, 16384 rows 16.6, 16.1; 1024 x 1024, 4096
// rows 14.9, 20.0, 8192 rows 26.9, 21.9; bf16 gradient of 512 x 512, 8192 rows 14.6, 19.9, 16384 rows 27.4, 21.4.
inline bool few_rows(const LinearArgs& a, bool streamed) {
    return a.n < 32768 && a.n * a.groups * a.steps < (streamed ? 1 << 20 : 1 << 19);
}

// Groups of features a workgroup of the resident kernel holds: as few feature blocks as LDS allows (each
// reads the rows again), the groups spread evenly over them (5 groups as 3 + 2 and not 4 + 1: every block
// gets the same share of the CUs); 0: not even one group fits.
inline int resident_groups(const LinearArgs& a) {
    int most = (kLdsBytes - channel_bytes<4>()) / (a.steps * 4096);
    if (most > 4) most = 4;
    if (most < 1) return 0;
    const int blocks = (a.groups + most - 1) / most;
    return (a.groups + blocks - 1) / blocks;
}

}  // namespace i8
}  // namespace nerf
