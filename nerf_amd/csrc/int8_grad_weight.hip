// nerf_linear_int8_grad_weight: dW[f][j] = sum over rows i of q[i][f] (s_i dz[i][j]) and db[j] = sum of
// dz[i][j], from the 8-bit rows a forward pass kept.  Formats: int8_common.h.
//
// The contraction runs over the rows, which lie far apart in memory for both operands: a stage of 32
// rows goes through registers into LDS as bf16 images [row][32 features] and is read back transposed
// (ds_read_b64_tr_b16) as the operands of v_mfma_f32_32x32x16_bf16.  An integer is exact in bf16; s_i, a
// power of two, moves only the exponent of dz, so dz times it is the exact sum of 1, 2 or 3 bf16 terms
// (bf16, fp16, fp32) and every product is exact; sums are fp32.
// A workgroup owns a tile of dW and a slice of the rows.  Slices are joined by a second kernel in slice
// order (no atomics: the same inputs give the same bits).
#include "int8_common.h"

namespace nerf {
namespace i8 {

typedef short short4v __attribute__((__vector_size__(4 * sizeof(short))));
typedef short short8 __attribute__((ext_vector_type(8)));

constexpr int kTileK = 128;       // input features of a workgroup's tile
constexpr int kStageRows = 32;
constexpr int kImg = kStageRows * 64;  // bytes of the image of 32 features: [32 rows][32 bf16]

struct GradWeightArgs {
    const signed char* q;
    const float* scale;
    const void* dz;
    int64_t n, lddz, rows_per;  // rows of a slice
    int k, kp, m, kblocks, mblocks, slices;
    float* out;                 // slice s: dW at out + s * stride
    float* out_db;              //          db at out_db + s * stride
    size_t stride;
};

// Operand (A or B) of 16 rows from an image: lane = feature (lane & 31), 8 rows from 8 (lane >> 5).
DEV bf16x8 tr_operand(const char* img, int half, int lane) {
    const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
    const char* base = img + (16 * half + 8 * (g >> 1) + q) * 64 + (g & 1) * 32 + p * 8;
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)base);
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(base + 4 * 64));
    const short8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8, v);
}

// EVEN: rows of dz are a whole number of 8-feature pieces, so that every piece is inside its row or wholly
// behind it (and then any piece of the row will do: its columns are not stored).
template <int DT, int MT, bool EVEN>
__global__ __launch_bounds__(256, 2) void grad_weight_kernel(GradWeightArgs a) {
    typedef typename Elem<DT>::T T;
    constexpr int N = Terms<DT>::N, YT = MT / 32, XT = kTileK / 32;
    constexpr int kChunks = MT >= 64 ? MT / 64 : 1;   // pieces of 8 features of dz per thread and stage
    constexpr int kStage = (XT + N * YT) * kImg;
    constexpr int AX = MT == 32 ? 1 : 2, AY = MT == 32 ? 1 : 2;  // 32 x 32 tiles of a wave
    constexpr int D = DT == NERF_F32 ? 2 : 4;  // even: the LDS buffer of a turn is then known when compiling
    static_assert(MT == 32 || MT == 128, "tile");
    __shared__ __attribute__((aligned(16))) char lds[2 * kStage];

    // workgroups 8 apart run on the same die and share its L2: the tiles of one slice read the same rows
    const int nb = a.kblocks * a.mblocks;
    int slice, blk;
    if (a.slices % 8 == 0) slice = (int)(blockIdx.x / 8 / nb) * 8 + (blockIdx.x & 7), blk = blockIdx.x / 8 % nb;
    else slice = blockIdx.x / nb, blk = blockIdx.x % nb;
    const int kb = blk % a.kblocks, mb = blk / a.kblocks;
    const int64_t lo = slice * a.rows_per;
    const int64_t hi = lo + a.rows_per < a.n ? lo + a.rows_per : a.n;
    const int64_t stages = hi > lo ? (hi - lo) / kStageRows : 0;  // whole ones; what is left is done last
    const int left = hi > lo ? (int)((hi - lo) % kStageRows) : 0;

    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // this thread's piece of the rows: 16 integers
    const int xh = t & 1, xt = (lane >> 4) & 3, xp = wave * 8 + ((lane >> 1) & 7);
    const int xcol = kb * kTileK + xt * 32 + xh * 16;
    // ... and of dz: 8 features of row yp, in the images yt0 + 2 i
    const int yq = t & 3, yp = (t >> 2) & 31, yt0 = t >> 7;
    const bool has_y = MT >= 64 || t < 128;

    const int xc = xcol < a.kp ? xcol : 0;   // columns behind the last are computed and not stored
    const bool y_whole = mb * MT + MT <= a.m;

    // Stages D - 1 turns ahead are on their way in registers: one stage of a workgroup is only some 12 KiB.
    struct Held {
        i32x4 x;
        Raw8<T> y[kChunks];
        float s;
    };
    Held held[D];
    float sum[kChunks][8];
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[i][j] = 0.f;

    // rows row0 + 0 .. 31; those behind `most` repeat it
    auto fetch = [&](int64_t row0, int64_t most, Held& h) {
        const int64_t rx = row0 + xp < most ? row0 + xp : most;
        h.x = *(const i32x4*)(a.q + rx * a.kp + xc);
        if (has_y) {
            const int64_t ry = row0 + yp < most ? row0 + yp : most;
            h.s = a.scale[ry];
            const T* src = (const T*)a.dz + ry * a.lddz;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int col = mb * MT + (yt0 + 2 * i) * 32 + yq * 8;
                if constexpr (EVEN) h.y[i] = load8<T>(src, col < a.m ? col : 0, a.m, true);
                else h.y[i] = load8<T>(src, col, a.m, y_whole);
            }
        }
    };
    auto stage = [&](const Held& h, char* buf, bool on) {
        {
            bf16x8 o[2];
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int b = 0; b < 4; ++b) o[w >> 1][(w & 1) * 4 + b] = (__bf16)(float)((h.x[w] << (24 - 8 * b)) >> 24);
            char* dst = buf + xt * kImg + xp * 64 + xh * 32;
            *(bf16x8*)dst = o[0];
            *(bf16x8*)(dst + 16) = o[1];
        }
        if (has_y) {
            const float xs = on ? h.s : 0.f;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                float v[8];
                to_float(h.y[i], v);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = on ? v[j] : 0.f;
                    sum[i][j] += v[j];
                    v[j] *= xs;
                }
                bf16x8 o[N];
                split_bf16<N>(v, o);
#pragma unroll
                for (int s = 0; s < N; ++s)
                    *(bf16x8*)(buf + (XT + s * YT + yt0 + 2 * i) * kImg + yp * 64 + yq * 16) = o[s];
            }
        }
    };

    const int wx = MT == 32 ? wave : 2 * (wave & 1), wy = MT == 32 ? 0 : 2 * (wave >> 1);
    f32x16 acc[AX][AY];
#pragma unroll
    for (int x = 0; x < AX; ++x)
#pragma unroll
        for (int y = 0; y < AY; ++y)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;

    auto multiply = [&](const char* buf) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            bf16x8 xo[AX];
#pragma unroll
            for (int x = 0; x < AX; ++x) xo[x] = tr_operand(buf + (wx + x) * kImg, half, lane);
#pragma unroll
            for (int s = 0; s < N; ++s)
#pragma unroll
                for (int y = 0; y < AY; ++y) {
                    const bf16x8 yo = tr_operand(buf + (XT + s * YT + wy + y) * kImg, half, lane);
#pragma unroll
                    for (int x = 0; x < AX; ++x) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xo[x], yo, acc[x][y], 0, 0, 0);
                }
        }
    };
    // every fetch is made, also of stages that do not exist (they repeat the last row): a wait for older
    // loads counts the younger ones
    if (hi > lo) {
#pragma unroll
        for (int d = 0; d < D; ++d) fetch(lo + d * kStageRows, hi - 1, held[d]);
        if (stages > 0) stage(held[0], lds, true);
        __syncthreads();
        for (int64_t st0 = 0; st0 < stages; st0 += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int64_t st = st0 + d;
                if (st >= stages) break;
                fetch(lo + (st + D) * kStageRows, hi - 1, held[d]);
                multiply(lds + (d & 1) * kStage);
                // into the buffer that was read in the turn before this one
                if (st + 1 < stages) stage(held[(d + 1) % D], lds + ((d + 1) & 1) * kStage, true);
                __syncthreads();
            }
        }
        if (left > 0) {
            fetch(lo + stages * kStageRows, hi - 1, held[0]);
            stage(held[0], lds, yp < left);
            __syncthreads();
            multiply(lds);
            __syncthreads();
        }
    }

    float* out = a.out + slice * a.stride;
#pragma unroll
    for (int x = 0; x < AX; ++x)
#pragma unroll
        for (int y = 0; y < AY; ++y) {
            const int col = mb * MT + (wy + y) * 32 + (lane & 31);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int f = kb * kTileK + (wx + x) * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
                if (f < a.k && col < a.m) out[(size_t)f * a.m + col] = acc[x][y][r];
            }
        }
    if (kb != 0) return;  // the whole workgroup
    // db: the 32 row lanes of a feature meet in LDS (free: behind the last barrier), added in row order
    float* red = (float*)lds;  // [32][MT]
    if (has_y) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) red[yp * MT + (yt0 + 2 * i) * 32 + yq * 8 + j] = sum[i][j];
    }
    __syncthreads();
    if (t < MT && mb * MT + t < a.m) {
        float s = 0.f;
        for (int p = 0; p < 32; ++p) s += red[p * MT + t];
        a.out_db[slice * a.stride + mb * MT + t] = s;
    }
}

// out[e] = sum over the slices of part[slice][e], in slice order within each of 8 runs of slices, the
// runs in order.  32 elements x 8 runs per workgroup: few elements (a head of 3 outputs) still load
// several slices at a time.
__global__ __launch_bounds__(256) void grad_weight_join_kernel(const float* __restrict__ part, int slices, size_t stride,
                                                               size_t n_dw, size_t count, float* __restrict__ dw,
                                                               float* __restrict__ db) {
    __shared__ float run[8][32];
    const size_t e = (size_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int r = threadIdx.x >> 5, per = (slices + 7) / 8;
    const int hi = (r + 1) * per < slices ? (r + 1) * per : slices;
    float s = 0.f;
    if (e < count) {
#pragma unroll 8
        for (int i = r * per; i < hi; ++i) s += part[(size_t)i * stride + e];
    }
    run[r][threadIdx.x & 31] = s;
    __syncthreads();
    if (threadIdx.x < 32 && e < count) {
        float v = run[0][threadIdx.x];
        for (int i = 1; i < 8; ++i) v += run[i][threadIdx.x];
        if (e < n_dw) dw[e] = v;
        else db[e - n_dw] = v;
    }
}

// How the rows are cut: enough slices for two workgroups per CU over all tiles, none under 256 rows.
struct Cut {
    int kblocks, mblocks, tile_m, slices;
    int64_t rows_per;
};
static Cut cut_rows(int64_t n, int k, int m) {
    Cut c;
    c.tile_m = m <= 32 ? 32 : 128;
    c.kblocks = (k + kTileK - 1) / kTileK, c.mblocks = (m + c.tile_m - 1) / c.tile_m;
    const int64_t blocks = (int64_t)c.kblocks * c.mblocks;
    int64_t s = 512 / blocks;
    const int64_t most = (n + 255) / 256;
    if (s > most) s = most;
    if (s >= 8) s = s / 8 * 8;
    if (s < 1) s = 1;
    c.slices = (int)s;
    c.rows_per = ((n + s - 1) / s + kStageRows - 1) / kStageRows * kStageRows;
    return c;
}

}  // namespace i8
}  // namespace nerf

using namespace nerf;
using namespace nerf::i8;

NERF_API size_t nerf_linear_int8_grad_weight_bytes(int64_t n, int k, int m) {
    if (n < 1 || k < 1 || m < 1 || k > kMaxWidth || m > kMaxWidth) return 0;
    const Cut c = cut_rows(n, k, m);
    return c.slices > 1 ? (size_t)c.slices * ((size_t)k + 1) * m * sizeof(float) : 0;
}

NERF_API int nerf_linear_int8_grad_weight(const signed char* q, const float* scale, int64_t n, int k, const void* dz,
                                          int dtype, int m, int64_t lddz, float* dw, float* db, void* workspace,
                                          size_t workspace_bytes, nerf_stream_t stream) {
    const char* what = "nerf_linear_int8_grad_weight";
    NERF_REQUIRE(n >= 1 && k >= 1 && m >= 1 && k <= kMaxWidth && m <= kMaxWidth, "%s: bad size (%lld rows, %d x %d)", what, (long long)n, k, m);
    NERF_REQUIRE(dtype_ok(dtype), "%s: unknown type %d", what, dtype);
    NERF_REQUIRE(q && scale && dz && dw && db, "%s: null pointer", what);
    NERF_REQUIRE(lddz >= m, "%s: rows overlap", what);
    NERF_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)dz & (dtype_size(dtype) - 1)) == 0 &&
                     (((uintptr_t)scale | (uintptr_t)dw | (uintptr_t)db | (uintptr_t)workspace) & 3) == 0,
                 "%s: misaligned pointer", what);
    const Cut c = cut_rows(n, k, m);
    const size_t need = nerf_linear_int8_grad_weight_bytes(n, k, m);
    NERF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: needs a workspace of %zu bytes, got %zu", what, need, workspace ? workspace_bytes : 0);
    GradWeightArgs a{};
    a.q = q, a.scale = scale, a.dz = dz, a.n = n, a.lddz = lddz, a.rows_per = c.rows_per;
    a.k = k, a.kp = (int)up64(k), a.m = m, a.kblocks = c.kblocks, a.mblocks = c.mblocks, a.slices = c.slices;
    const size_t n_dw = (size_t)k * m;
    if (c.slices > 1) a.out = (float*)workspace, a.out_db = (float*)workspace + n_dw, a.stride = n_dw + m;
    else a.out = dw, a.out_db = db, a.stride = 0;
    const unsigned grid = (unsigned)((int64_t)c.kblocks * c.mblocks * c.slices);
    hipStream_t st = as_stream(stream);
#define NERF_W(DT)                                                                     \
    do {                                                                               \
        if (c.tile_m == 32) grad_weight_kernel<DT, 32, false><<<grid, 256, 0, st>>>(a);     \
        else if (m % 8 == 0) grad_weight_kernel<DT, 128, true><<<grid, 256, 0, st>>>(a);    \
        else grad_weight_kernel<DT, 128, false><<<grid, 256, 0, st>>>(a);                   \
    } while (0)
    if (dtype == NERF_F32) NERF_W(NERF_F32);
    else if (dtype == NERF_F16) NERF_W(NERF_F16);
    else NERF_W(NERF_BF16);
#undef NERF_W
    if (int rc = check_launch(what)) return rc;
    if (c.slices > 1) {
        grad_weight_join_kernel<<<(unsigned)((n_dw + m + 31) / 32), 256, 0, st>>>((const float*)workspace, c.slices, a.stride, n_dw, n_dw + m, dw, db);
        return check_launch(what);
    }
    return 0;
}
