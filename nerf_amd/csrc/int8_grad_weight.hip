// nerf_linear_int8_grad_weight: dW[f][j] = sum over rows i of q[i][f] (s_i dz[i][j]) and db[j] = sum of
// dz[i][j], from the 8-bit rows a forward pass kept.  Formats: int8_common.h.
//
// The contraction runs over the rows, which lie far apart in memory for both operands: a stage of 32 or 64
// rows goes through registers into LDS as bf16 images [row][32 features] and is read back transposed
// (ds_read_b64_tr_b16) as the operands of v_mfma_f32_32x32x16_bf16.  An integer times s_i, a power of two, is
// exact in bf16 (the scale goes with the integers: bf16 dz then passes untouched), dz is the exact sum
// of 1, 2 or 3 bf16 terms (bf16, fp16, fp32), so every product is exact; sums are fp32.
// A workgroup owns a tile of dW and a slice of the rows.  Slices are joined by a second kernel in slice
// order (no atomics: the same inputs give the same bits).
// Bound by memory where the tiles cover dW (786432 x 256 x 256 bf16: 133 us, 5.1 TB/s of rows and partial
// sums, + 11 us for the join); fp32 dz by its three products.
#include "int8_common.h"

namespace nerf {
namespace i8 {

typedef short short4v __attribute__((__vector_size__(4 * sizeof(short))));
typedef short short8 __attribute__((ext_vector_type(8)));

struct GradWeightArgs {
    const signed char* q;
    const float* scale;
    const void* dz;
    int64_t n, lddz, rows_per;  // rows of a slice
    int k, kp, m, kblocks, mblocks, slices;  // blocks: of the tile's features
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

// KT x MT features of dW by four waves (256 x 256: eight), stages of R rows, D of them held ahead in registers (even: the LDS
// buffer of a turn is then known when compiling).
// EVEN: rows of dz are a whole number of 8-feature pieces, so that every piece is inside its row or wholly
// behind it (and then any piece of the row will do: its columns are not stored).
template <int DT, int KT, int MT, int R, int D, bool EVEN>
__global__ __launch_bounds__(KT == 256 ? 512 : 256, 2) void grad_weight_kernel(GradWeightArgs a) {
    constexpr int NT = KT == 256 ? 512 : 256;  // threads
    typedef typename Elem<DT>::T T;
    constexpr int N = Terms<DT>::N, YT = MT / 32, XT = KT / 32;
    constexpr int kImg = R * 64;  // bytes of the image of 32 features: [R rows][32 bf16]
    constexpr int kStage = (XT + N * YT) * kImg;
    constexpr int kXPieces = R * KT / 16, kYPieces = R * MT / 8;   // 16 integers, 8 elements of dz
    constexpr int CX = (kXPieces + NT - 1) / NT, CY = (kYPieces + NT - 1) / NT;  // of a thread
    // waves along k and m, and 32 x 32 tiles of a wave
    constexpr int WX = MT == 32 ? 4 : KT >= 128 ? 2 : 1, WY = NT / 64 / WX, AX = XT / WX, AY = YT / WY;
    constexpr int kRowBits = R == 64 ? 6 : 5, kTileBits = KT == 256 ? 3 : KT == 128 ? 2 : 1;
    static_assert((R == 32 || R == 64) && (KT == 64 || KT == 128 || KT == 256) && AX >= 1 && AY >= 1 && D % 2 == 0, "shapes");
    __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
    static_assert(2 * kStage >= R * MT * 4, "the sums of dz meet in LDS");

    // workgroups 8 apart run on the same die and share its L2: the tiles of one slice read the same rows
    const int nb = a.kblocks * a.mblocks;
    int slice, blk;
    if (a.slices % 8 == 0) slice = (int)(blockIdx.x / 8 / nb) * 8 + (blockIdx.x & 7), blk = blockIdx.x / 8 % nb;
    else slice = blockIdx.x / nb, blk = blockIdx.x % nb;
    const int kb = blk % a.kblocks, mb = blk / a.kblocks;
    const int64_t lo = slice * a.rows_per;
    const int64_t hi = lo + a.rows_per < a.n ? lo + a.rows_per : a.n;
    const int64_t stages = hi > lo ? (hi - lo) / R : 0;  // whole ones; what is left is done last
    const int left = hi > lo ? (int)((hi - lo) % R) : 0;

    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // Piece e of the rows: half of an image's 32 features (bit 0), 3 bits of the row, the image, the other bits of
    // the row: a wave reads runs of a row and writes LDS without conflicts.  Piece e of dz: a quarter of an
    // image (2 bits), the row, the image.
    auto x_half = [&](int e) { return e & 1; };
    auto x_img = [&](int e) { return (e >> 4) & (XT - 1); };
    auto x_row = [&](int e) { return ((e >> 1) & 7) | (e >> (4 + kTileBits)) << 3; };
    auto y_row = [&](int e) { return (e >> 2) & (R - 1); };
    auto y_img = [&](int e) { return e >> (2 + kRowBits); };
    const int yq = t & 3;
    const bool has_x = kXPieces >= NT || t < kXPieces, has_y = kYPieces >= NT || t < kYPieces;
    const bool y_whole = mb * MT + MT <= a.m;

    struct Held {
        i32x4 x[CX];
        float s[CX];
        Raw8<T> y[CY];
    };
    Held held[D];
    float sum[CY][8];
#pragma unroll
    for (int i = 0; i < CY; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[i][j] = 0.f;

    // Where a thread's pieces are, from the first row of a stage: the same for every stage, so that a fetch is a
    // scalar base and these.
    unsigned x_at[CX], s_at[CX];
    int64_t y_at[CY];
#pragma unroll
    for (int i = 0; i < CX; ++i) {
        const int e = t + NT * i, col = kb * KT + x_img(e) * 32 + x_half(e) * 16;
        x_at[i] = (unsigned)x_row(e) * a.kp + (col < a.kp ? col : 0);  // (behind the last column: not stored)
        s_at[i] = x_row(e);
    }
    auto y_col = [&](int i) {
        const int col = mb * MT + y_img(t + NT * i) * 32 + yq * 8;
        return EVEN && col >= a.m ? 0 : col;
    };
#pragma unroll
    for (int i = 0; i < CY; ++i) y_at[i] = y_row(t + NT * i) * a.lddz;
    // the stage from row0, which has rows at least up to row0 + `most`; rows behind repeat that one
    auto fetch = [&](int64_t row0, int most, Held& h) {
        if (has_x) {
            const signed char* q = a.q + row0 * a.kp;
            const float* sc = a.scale + row0;
#pragma unroll
            for (int i = 0; i < CX; ++i) {
                const unsigned back = (int)s_at[i] > most ? s_at[i] - most : 0u;
                h.x[i] = *(const i32x4*)(q + (x_at[i] - back * a.kp));
                h.s[i] = sc[s_at[i] - back];
            }
        }
        if (has_y) {
            const T* y = (const T*)a.dz + row0 * a.lddz;
#pragma unroll
            for (int i = 0; i < CY; ++i) {
                const int row = y_row(t + NT * i);
                const T* src = y + (y_at[i] - (row > most ? (row - most) * a.lddz : 0));
                h.y[i] = load8<T>(src, y_col(i), a.m, EVEN || y_whole);
            }
        }
    };
    // ... into LDS as bf16; of a last stage only the first `rows`
    auto stage = [&](const Held& h, char* buf, int rows) {
        if (has_x) {
#pragma unroll
            for (int i = 0; i < CX; ++i) {
                const int e = t + NT * i;
                const float xs = x_row(e) < rows ? h.s[i] : 0.f;
                bf16x8 o[2];
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                    for (int b = 0; b < 4; ++b) o[w >> 1][(w & 1) * 4 + b] = (__bf16)((float)((h.x[i][w] << (24 - 8 * b)) >> 24) * xs);
                char* dst = buf + x_img(e) * kImg + x_row(e) * 64 + x_half(e) * 32;
                *(bf16x8*)dst = o[0];
                *(bf16x8*)(dst + 16) = o[1];
            }
        }
        if (has_y) {
#pragma unroll
            for (int i = 0; i < CY; ++i) {
                const int e = t + NT * i;
                const bool on = y_row(e) < rows;
                bf16x8 o[N];
                if (DT != NERF_BF16 || kb == 0) {
                    float v[8];
                    to_float(h.y[i], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[j] = on ? v[j] : 0.f;
                        sum[i][j] += v[j];
                    }
                    if constexpr (DT != NERF_BF16) split_bf16<N>(v, o);
                }
                if constexpr (DT == NERF_BF16) o[0] = __builtin_bit_cast(bf16x8, on ? h.y[i].w[0] : i32x4{0, 0, 0, 0});
#pragma unroll
                for (int s = 0; s < N; ++s) *(bf16x8*)(buf + (XT + s * YT + y_img(e)) * kImg + y_row(e) * 64 + yq * 16) = o[s];
            }
        }
    };

    const int wx = (wave % WX) * AX, wy = (wave / WX) * AY;
    f32x16 acc[AX][AY];
#pragma unroll
    for (int x = 0; x < AX; ++x)
#pragma unroll
        for (int y = 0; y < AY; ++y)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;
    // 16 rows at a time; the operands of the next 16 are read before the products of these (left to itself the
    // compiler reads right before use, and every product waits for LDS)
    struct Operands {
        bf16x8 x[AX], y[N][AY];
    };
    auto read = [&](const char* buf, int half, Operands& o) {
#pragma unroll
        for (int x = 0; x < AX; ++x) o.x[x] = tr_operand(buf + (wx + x) * kImg, half, lane);
#pragma unroll
        for (int s = 0; s < N; ++s)
#pragma unroll
            for (int y = 0; y < AY; ++y) o.y[s][y] = tr_operand(buf + (XT + s * YT + wy + y) * kImg, half, lane);
    };
    auto products = [&](const Operands& c) {
#pragma unroll
        for (int s = 0; s < N; ++s)
#pragma unroll
            for (int y = 0; y < AY; ++y)
#pragma unroll
                for (int x = 0; x < AX; ++x) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(c.x[x], c.y[s][y], acc[x][y], 0, 0, 0);
    };
    auto multiply = [&](const char* buf) {
        if constexpr (KT == 256) {  // (no room for two sets)
#pragma unroll
            for (int half = 0; half < R / 16; ++half) {
                Operands o;
                read(buf, half, o);
                products(o);
            }
        } else {
            Operands o[2];
            read(buf, 0, o[0]);
#pragma unroll
            for (int half = 0; half < R / 16; ++half) {
                if (half + 1 < R / 16) read(buf, half + 1, o[(half + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
                products(o[half & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // every fetch is made, also of stages that do not exist (they repeat the last): a wait for older loads
    // counts the younger ones
    if (stages > 0) {
        auto fetch_whole = [&](int64_t st, Held& h) { fetch(lo + (st < stages ? st : stages - 1) * R, R - 1, h); };
#pragma unroll
        for (int d = 0; d < D; ++d) fetch_whole(d, held[d]);
        stage(held[0], lds, R);
        __syncthreads();
        for (int64_t st0 = 0; st0 < stages; st0 += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int64_t st = st0 + d;
                if (st >= stages) break;
                fetch_whole(st + D, held[d]);
                multiply(lds + (d & 1) * kStage);
                // into the buffer that was read in the turn before this one
                if (st + 1 < stages) stage(held[(d + 1) % D], lds + ((d + 1) & 1) * kStage, R);
                __syncthreads();
            }
        }
    }
    if (left > 0) {
        fetch(lo + stages * R, left - 1, held[0]);
        stage(held[0], lds, left);
        __syncthreads();
        multiply(lds);
        __syncthreads();
    }

    float* out = a.out + slice * a.stride;
#pragma unroll
    for (int x = 0; x < AX; ++x)
#pragma unroll
        for (int y = 0; y < AY; ++y) {
            const int col = mb * MT + (wy + y) * 32 + (lane & 31);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int f = kb * KT + (wx + x) * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
                if (f < a.k && col < a.m) out[(size_t)f * a.m + col] = acc[x][y][r];
            }
        }
    if (kb != 0) return;  // the whole workgroup
    // db: the row lanes of a feature meet in LDS (free: behind the last barrier), added in row order
    float* red = (float*)lds;  // [R][MT]
    if (has_y) {
#pragma unroll
        for (int i = 0; i < CY; ++i) {
            const int e = t + NT * i;
#pragma unroll
            for (int j = 0; j < 8; ++j) red[y_row(e) * MT + y_img(e) * 32 + yq * 8 + j] = sum[i][j];
        }
    }
    __syncthreads();
    if (t < MT && mb * MT + t < a.m) {
        float s = 0.f;
        for (int p = 0; p < R; ++p) s += red[p * MT + t];
        a.out_db[slice * a.stride + mb * MT + t] = s;
    }
}

// Up to four outputs (the colour and density heads): a matrix tile would be nearly empty, so a thread owns 16
// input features, streams its share of the rows past 16 M sums in registers (one conversion and M
// multiply-adds an integer, which the rows' bytes still outlast) and the workgroup's threads meet in LDS
// at the end.  blockIdx.y: blocks of 64 pieces of 16 features.
constexpr int kThinPieces = 64;
template <int DT, int M>
__global__ __launch_bounds__(256) void grad_weight_thin_kernel(GradWeightArgs a) {
    typedef typename Elem<DT>::T T;
    __shared__ float lds[256 * 16 * M];
    __shared__ float lds_db[256 * M];
    const int t = threadIdx.x;
    const int p0 = blockIdx.y * kThinPieces, all = a.kp / 16;
    const int pieces = all - p0 < kThinPieces ? all - p0 : kThinPieces, lanes = 256 / pieces;  // rows side by side
    const int c = t % pieces, rl = t / pieces;
    const int64_t lo = blockIdx.x * a.rows_per;
    const int64_t hi = lo + a.rows_per < a.n ? lo + a.rows_per : a.n;
    float acc[M][16], db[M];
#pragma unroll
    for (int j = 0; j < M; ++j) {
        db[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[j][i] = 0.f;
    }
    constexpr int U = 8;  // rows of a thread on their way at a time (786432 x 128 x 3: 36 us, with four 40)
    if (rl < lanes && hi > lo) {
        const signed char* q = a.q + (p0 + c) * 16;
        for (int64_t row0 = lo + rl; row0 < hi; row0 += U * lanes) {
            i32x4 x[U];
            float s[U], d[U][M];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = row0 + u * lanes < hi ? row0 + u * lanes : hi - 1;
                x[u] = *(const i32x4*)(q + row * a.kp);
                s[u] = a.scale[row];
#pragma unroll
                for (int j = 0; j < M; ++j) d[u][j] = (float)((const T*)a.dz)[row * a.lddz + j];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool on = row0 + u * lanes < hi;
#pragma unroll
                for (int j = 0; j < M; ++j) {
                    d[u][j] = on ? d[u][j] : 0.f;
                    db[j] += d[u][j];
                    d[u][j] *= on ? s[u] : 0.f;
                }
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const float v = (float)((x[u][w] << (24 - 8 * b)) >> 24);
#pragma unroll
                        for (int j = 0; j < M; ++j) acc[j][4 * w + b] = __builtin_fmaf(v, d[u][j], acc[j][4 * w + b]);
                    }
            }
        }
    }
    if (rl < lanes) {
#pragma unroll
        for (int j = 0; j < M; ++j) {
            if (c == 0) lds_db[rl * M + j] = db[j];
#pragma unroll
            for (int i = 0; i < 16; ++i) lds[((rl * pieces + c) * 16 + i) * M + j] = acc[j][i];
        }
    }
    __syncthreads();
    for (int e = t; e < pieces * 16 * M; e += 256) {
        float s = 0.f;
        for (int r = 0; r < lanes; ++r) s += lds[r * pieces * 16 * M + e];
        const int f = p0 * 16 + e / M;
        if (f < a.k) a.out[blockIdx.x * a.stride + (size_t)f * M + e % M] = s;
    }
    if (blockIdx.y == 0 && t < M) {
        float s = 0.f;
        for (int r = 0; r < lanes; ++r) s += lds_db[r * M + t];
        a.out_db[blockIdx.x * a.stride + t] = s;
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

// Which tiles, and how the rows are cut: up to `target` workgroups over all tiles, slices of at least 256 rows,
// for few outputs eight rows a thread (206602 x 27 x 3: 21 us, with slices of 256 rows 29; 4000 x 256 x 3: 15.5, 16).
// bf16 tiles of 256 x 256, one workgroup a CU, read every row once (of 128 x 128: from L2 by two workgroups), but
// leave twice the partial sums to join.  They are taken where they waste no more than those of 128 and where
// slices have 2048 rows or more: 786432 x 256 x 256 133 + 11 us (of 128: 144 + 6; memory at the rate of a copy),
// 262144 x 512 x 256 100 us in all (104), 65536 x 256 x 256 41 us (32).
struct Cut {
    int tile_k, tile_m;  // tile_m 0: the kernel for few outputs
    int kblocks, mblocks, slices;
    int64_t rows_per;
};
static Cut cut_rows(int64_t n, int k, int m, bool bf16) {
    Cut c;
    const bool thin = m <= 4;
    const auto blocks_of = [](int size, int tile) { return (size + tile - 1) / tile; };
    const int k256 = blocks_of(k, 256), m256 = blocks_of(m, 256);
    const bool wide = bf16 && m % 8 == 0 && 2 * k256 == blocks_of(k, 128) && 2 * m256 == blocks_of(m, 128) && n * k256 * m256 >= 256 * 2048;
    c.tile_m = thin ? 0 : m <= 32 ? 32 : wide ? 256 : 128;
    c.tile_k = thin ? kThinPieces * 16 : wide ? 256 : (m > 32 && k <= 64) ? 64 : 128;
    c.kblocks = blocks_of(k, c.tile_k), c.mblocks = thin ? 1 : blocks_of(m, c.tile_m);
    const int64_t blocks = (int64_t)c.kblocks * c.mblocks;
    const int64_t target = wide ? 256 : c.tile_m == 128 ? 512 : 1024;  // as many a CU as their registers allow
    int64_t s = target / blocks;
    const int pieces = (int)up64(k) / 16;
    const int least = !thin ? 256 : pieces < 32 ? 2048 / pieces : 64;
    const int64_t most = (n + least - 1) / least;
    if (s > most) s = most;
    if (s >= 8) s = s / 8 * 8;
    if (s < 1) s = 1;
    c.slices = (int)s;
    c.rows_per = ((n + s - 1) / s + 63) / 64 * 64;
    return c;
}

template <int DT>
static void launch_grad_weight(const GradWeightArgs& a, const Cut& c, hipStream_t st) {
    if (c.tile_m == 0) {
        const dim3 grid(c.slices, c.kblocks);
        if (a.m == 1) grad_weight_thin_kernel<DT, 1><<<grid, 256, 0, st>>>(a);
        else if (a.m == 2) grad_weight_thin_kernel<DT, 2><<<grid, 256, 0, st>>>(a);
        else if (a.m == 3) grad_weight_thin_kernel<DT, 3><<<grid, 256, 0, st>>>(a);
        else grad_weight_thin_kernel<DT, 4><<<grid, 256, 0, st>>>(a);
        return;
    }
    const unsigned grid = (unsigned)((int64_t)c.kblocks * c.mblocks * c.slices);
    constexpr int D = DT == NERF_F32 ? 2 : 4;
    const bool even = a.m % 8 == 0;
    if (c.tile_m == 256) grad_weight_kernel<NERF_BF16, 256, 256, 32, 4, true><<<grid, 512, 0, st>>>(a);
    else if (c.tile_m == 32) grad_weight_kernel<DT, 128, 32, 32, 4, false><<<grid, 256, 0, st>>>(a);
    else if (c.tile_k == 64) {
        if (even) grad_weight_kernel<DT, 64, 128, 32, D, true><<<grid, 256, 0, st>>>(a);
        else grad_weight_kernel<DT, 64, 128, 32, D, false><<<grid, 256, 0, st>>>(a);
    } else {
        // (stages of 64 rows where LDS holds two of them twice over: 786432 x 256 x 256, 198 -> 182 us)
        if (even && DT == NERF_BF16) grad_weight_kernel<DT, 128, 128, DT == NERF_BF16 ? 64 : 32, 2, true><<<grid, 256, 0, st>>>(a);
        else if (even) grad_weight_kernel<DT, 128, 128, 32, D, true><<<grid, 256, 0, st>>>(a);
        else grad_weight_kernel<DT, 128, 128, 32, D, false><<<grid, 256, 0, st>>>(a);
    }
}

}  // namespace i8
}  // namespace nerf

using namespace nerf;
using namespace nerf::i8;

NERF_API size_t nerf_linear_int8_grad_weight_bytes(int64_t n, int k, int m) {
    if (n < 1 || k < 1 || m < 1 || k > kMaxWidth || m > kMaxWidth) return 0;
    const int s = cut_rows(n, k, m, false).slices, t = cut_rows(n, k, m, true).slices, slices = s > t ? s : t;
    return slices > 1 ? (size_t)slices * ((size_t)k + 1) * m * sizeof(float) : 0;
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
    const Cut c = cut_rows(n, k, m, dtype == NERF_BF16);
    const size_t need = nerf_linear_int8_grad_weight_bytes(n, k, m);
    NERF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: needs a workspace of %zu bytes, got %zu", what, need, workspace ? workspace_bytes : 0);
    GradWeightArgs a{};
    a.q = q, a.scale = scale, a.dz = dz, a.n = n, a.lddz = lddz, a.rows_per = c.rows_per;
    a.k = k, a.kp = (int)up64(k), a.m = m, a.kblocks = c.kblocks, a.mblocks = c.mblocks, a.slices = c.slices;
    const size_t n_dw = (size_t)k * m;
    if (c.slices > 1) a.out = (float*)workspace, a.out_db = (float*)workspace + n_dw, a.stride = n_dw + m;
    else a.out = dw, a.out_db = db, a.stride = 0;
    hipStream_t st = as_stream(stream);
    if (dtype == NERF_F32) launch_grad_weight<NERF_F32>(a, c, st);
    else if (dtype == NERF_F16) launch_grad_weight<NERF_F16>(a, c, st);
    else launch_grad_weight<NERF_BF16>(a, c, st);
    if (int rc = check_launch(what)) return rc;
    if (c.slices > 1) {
        grad_weight_join_kernel<<<(unsigned)((n_dw + m + 31) / 32), 256, 0, st>>>((const float*)workspace, c.slices, a.stride, n_dw, n_dw + m, dw, db);
        return check_launch(what);
    }
    return 0;
}
