// Rows and weights in 8-bit integers: nerf_quantize_rows, nerf_int8_pack.  Formats: int8_common.h.
#include "int8_common.h"

namespace nerf {
namespace i8 {

// One row by `tpr` neighbouring lanes (a power of two, at most a wave): each holds NV pieces of 8
// neighbouring elements, the largest magnitude is exchanged between the lanes, the integers leave as
// 8-byte stores and the bits as one byte per piece.  NV = 0: rows too long for registers are read
// twice (the second time mostly out of L2).  Bound by memory: reads the row once, writes kp + 4
// (+ kp / 8) bytes.
template <int DT, int NV>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* __restrict__ xv, int64_t n, int k, int64_t ldx,
                                                            int pow2, int tpr, signed char* __restrict__ q,
                                                            float* __restrict__ scale, unsigned char* __restrict__ mask) {
    typedef typename Elem<DT>::T T;
    const int lane = threadIdx.x & (tpr - 1);
    const int kp = (int)up64(k), pieces = kp / 8;
    for (int64_t row = (int64_t)blockIdx.x * (256 / tpr) + threadIdx.x / tpr; row < n; row += (int64_t)gridDim.x * (256 / tpr)) {
        const T* x = (const T*)xv + row * ldx;
        unsigned top = 0u;
        float v[NV > 0 ? NV : 1][8];
        auto read = [&](int c, float (&w)[8]) {
            load_row<T, 8>(x + 8 * c, k - 8 * c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned a = magnitude(w[i]);
                top = top > a ? top : a;
            }
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (lane + j * tpr < pieces) read(lane + j * tpr, v[j]);
        } else {
            for (int c = lane; c < pieces; c += tpr) read(c, v[0]);
        }
        for (int off = tpr >> 1; off > 0; off >>= 1) {  // the lanes of a row are all here or all gone
            const unsigned o = (unsigned)__shfl_xor((int)top, off);
            top = top > o ? top : o;
        }
        const Scale sc = scale_of(top, pow2 != 0);
        if (lane == 0) scale[row] = sc.scale;
        signed char* qr = q + row * kp;
        unsigned char* mr = mask ? mask + row * (kp / 8) : nullptr;
        auto write = [&](int c, const float (&w)[8]) {
            float lo[4], hi[4];
            unsigned bits = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) lo[i] = w[i] * sc.inv + kRoundAt, hi[i] = w[i + 4] * sc.inv + kRoundAt;
#pragma unroll
            for (int i = 0; i < 8; ++i) bits |= w[i] > 0.f ? 1u << i : 0u;
            *(uint2*)(qr + 8 * c) = sc.inv == 0.f ? make_uint2(0u, 0u) : make_uint2(low_bytes(lo), low_bytes(hi));
            if (mr) mr[c] = (unsigned char)bits;
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (lane + j * tpr < pieces) write(lane + j * tpr, v[j]);
        } else {
            for (int c = lane; c < pieces; c += tpr) {
                float w[8];
                load_row<T, 8>(x + 8 * c, k - 8 * c, w);
                write(c, w);
            }
        }
    }
}

// One workgroup per group of 64 output channels (x) and share of the input rows (y): the channels'
// largest magnitudes over all rows of W, then its share of the fragments.  Every workgroup of a
// channel group forms the same scales (W is small and in L2), so that none waits for another.
constexpr int kPackThreads = 1024;
__global__ __launch_bounds__(kPackThreads) void int8_pack_kernel(const float* __restrict__ w, int k, int m, int pow2,
                                                                 char* __restrict__ packed, PackedLayout lay) {
    __shared__ unsigned part[kPackThreads / 64][64];
    __shared__ float s_scale[64], s_inv[64];
    const int t = threadIdx.x, T = blockIdx.x;
    {
        const int j = 64 * T + (t & 63);
        unsigned top = 0u;
        if (j < m) {
#pragma unroll 8
            for (int f = t >> 6; f < k; f += kPackThreads / 64) {
                const unsigned a = magnitude(w[(size_t)f * m + j]);
                top = top > a ? top : a;
            }
        }
        part[t >> 6][t & 63] = top;
    }
    __syncthreads();
    if (t < 64) {
        unsigned top = 0u;
        for (int i = 0; i < kPackThreads / 64; ++i) top = top > part[i][t] ? top : part[i][t];
        Scale sc = scale_of(top, pow2 != 0);
        if (64 * T + t >= m) sc.scale = 0.f;  // no such channel
        s_scale[t] = sc.scale, s_inv[t] = sc.inv;
        if (blockIdx.y == 0) ((float*)packed)[64 * T + t] = sc.scale;
    }
    __syncthreads();
    const int ksteps = lay.kp / 64, msteps = lay.mp / 32;
    const int lane = t & 63, u = (t >> 6) & 3, r = lane & 15, g = lane >> 4;
    // a step of 64 inputs per turn of the workgroup: 256 threads the integers, one 16-byte piece each, and with
    // pow2 512 more the transposed copy in bf16 (two steps of 32 channels of this group)
    const int part_of = t >> 8;
    for (int s = blockIdx.y; s < ksteps; s += gridDim.y) {
        if (part_of == 0) {
            const int c = frag_feature(u, r), j = 64 * T + c, f0 = 64 * s + 16 * g;
            unsigned o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int e[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int f = f0 + 4 * i + b;
                    e[b] = (j < m && f < k) ? quantised(w[(size_t)f * m + j], s_inv[c]) : 0;
                }
                o[i] = pack4(e[0], e[1], e[2], e[3]);
            }
            *(uint4*)(packed + lay.frags + ((((size_t)T * ksteps + s) * 4 + u) * 64 + lane) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
        } else if (pow2 && part_of < 3) {
            const int half = part_of - 1, c0 = 32 * half + 8 * g, f = 64 * s + frag_feature(u, r);
            bf16x8 o;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 64 * T + c0 + i;
                o[i] = (j < m && f < k) ? (__bf16)((float)quantised(w[(size_t)f * m + j], s_inv[c0 + i]) * s_scale[c0 + i]) : (__bf16)0.f;
            }
            *(bf16x8*)(packed + lay.frags_t + ((((size_t)s * msteps + 2 * T + half) * 4 + u) * 64 + lane) * 16) = o;
        }
    }
}

}  // namespace i8
}  // namespace nerf

using namespace nerf;
using namespace nerf::i8;

NERF_API size_t nerf_int8_packed_bytes(int k, int m, int pow2) {
    if (k < 1 || m < 1 || k > kMaxWidth || m > kMaxWidth) return 0;
    return PackedLayout(k, m, pow2 != 0).bytes;
}

NERF_API int nerf_int8_pack(const float* w, int k, int m, int pow2, void* packed, nerf_stream_t stream) {
    NERF_REQUIRE(w && packed, "nerf_int8_pack: null pointer");
    NERF_REQUIRE(k >= 1 && m >= 1 && k <= kMaxWidth && m <= kMaxWidth, "nerf_int8_pack: widths must be in [1, %d], got %d x %d", kMaxWidth, k, m);
    NERF_REQUIRE(((uintptr_t)packed & 15) == 0 && ((uintptr_t)w & 3) == 0, "nerf_int8_pack: misaligned pointer");
    const PackedLayout lay(k, m, pow2 != 0);
    const int steps = lay.kp / 64;
    const dim3 grid(lay.mp / 64, steps < 32 ? steps : 32);  // a step of 64 inputs each where there are that few
    int8_pack_kernel<<<grid, kPackThreads, 0, as_stream(stream)>>>(w, k, m, pow2, (char*)packed, lay);
    return check_launch("nerf_int8_pack");
}

template <int DT>
static void launch_quantize(const void* x, int64_t n, int k, int64_t ldx, int pow2, signed char* q, float* scale,
                            unsigned char* mask, hipStream_t st) {
    const int pieces = (int)up64(k) / 8;
    int tpr = 8;
    while (tpr < pieces && tpr < 64) tpr *= 2;
    const int per = (pieces + tpr - 1) / tpr;
    const int64_t want = (n + 256 / tpr - 1) / (256 / tpr);
    const unsigned blocks = (unsigned)(want < (1 << 22) ? want : (1 << 22));  // a launch holds fewer than 2^32 work items
#define NERF_Q(NV) quantize_rows_kernel<DT, NV><<<blocks, 256, 0, st>>>(x, n, k, ldx, pow2, tpr, q, scale, mask)
    if (per <= 1) NERF_Q(1);
    else if (per <= 2) NERF_Q(2);
    else if (per <= 4) NERF_Q(4);
    else NERF_Q(0);
#undef NERF_Q
}

NERF_API int nerf_quantize_rows(const void* x, int dtype, int64_t n, int k, int64_t ldx, int pow2, signed char* q,
                                float* scale, unsigned char* mask, nerf_stream_t stream) {
    NERF_REQUIRE(n >= 0 && k >= 1 && k <= kMaxWidth, "nerf_quantize_rows: bad size (%lld x %d)", (long long)n, k);
    NERF_REQUIRE(dtype_ok(dtype), "nerf_quantize_rows: unknown type %d", dtype);
    if (n == 0) return 0;
    NERF_REQUIRE(x && q && scale, "nerf_quantize_rows: null pointer");
    NERF_REQUIRE(ldx >= k, "nerf_quantize_rows: rows of %d elements overlap at a distance of %lld", k, (long long)ldx);
    NERF_REQUIRE((((uintptr_t)q) & 15) == 0 && ((uintptr_t)x & (dtype_size(dtype) - 1)) == 0 && ((uintptr_t)scale & 3) == 0,
                 "nerf_quantize_rows: misaligned pointer");
    hipStream_t st = as_stream(stream);
    if (dtype == NERF_F32) launch_quantize<NERF_F32>(x, n, k, ldx, pow2, q, scale, mask, st);
    else if (dtype == NERF_F16) launch_quantize<NERF_F16>(x, n, k, ldx, pow2, q, scale, mask, st);
    else launch_quantize<NERF_BF16>(x, n, k, ldx, pow2, q, scale, mask, st);
    return check_launch("nerf_quantize_rows");
}
