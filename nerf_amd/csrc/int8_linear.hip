// nerf_linear_int8, nerf_linear_int8_quantized: rows in 8-bit integers times weights in 8-bit integers.
#include "int8_product.h"

namespace nerf {
namespace i8 {

// Groups of 64 channels up to which a row of 8-bit output is one workgroup's.
constexpr int kRowGroups = 8;

// Tiles of 16 points a wave works on at a time: two halve the reads of LDS and of the channel scales, where
// the registers hold the sums of both.
template <int OUT, int NT, int CH, int ADD>
constexpr int kTiles = (NT == 4 && (CH > 4 || ADD != NO_ADD || OUT >= TO_INT8)) || (NT == 2 && ADD != NO_ADD && OUT >= TO_INT8) ? 1 : 2;

template <int OUT, int NT, int ADD>
static int resident(const LinearArgs& a, const char* what, hipStream_t st) {
    // all of a row in one unit up to 320 inputs (beside an addend's memory traffic a step read twice costs little)
    if constexpr (ADD != NO_ADD) return launch_resident<Int8Op, OUT, NT, 4, kTiles<OUT, NT, 4, ADD>, ADD>(a, what, st);
    else switch (a.steps) {
        case 1: return launch_resident<Int8Op, OUT, NT, 1, kTiles<OUT, NT, 1, ADD>, ADD>(a, what, st);
        case 2: return launch_resident<Int8Op, OUT, NT, 2, kTiles<OUT, NT, 2, ADD>, ADD>(a, what, st);
        case 5: return launch_resident<Int8Op, OUT, NT, 5, kTiles<OUT, NT, 5, ADD>, ADD>(a, what, st);
        case 3: case 6: case 9: return launch_resident<Int8Op, OUT, NT, 3, kTiles<OUT, NT, 3, ADD>, ADD>(a, what, st);
        default: return launch_resident<Int8Op, OUT, NT, 4, kTiles<OUT, NT, 4, ADD>, ADD>(a, what, st);
    }
}

template <int OUT, int ADD>
static int launch(const LinearArgs& a, const char* what, hipStream_t st) {
    const int nt = a.groups == 3 ? 4 : a.groups;  // (of three groups' kernel one would be idle)
    const bool fits = nt <= 4 && channel_bytes<4>() + (int64_t)nt * a.steps * 4096 <= kLdsBytes;
    if constexpr (OUT < TO_INT8) {
        if (few_rows(a, !fits)) return launch_direct<Int8Op, OUT, ADD>(a, what, st);
        if (!fits) return launch_streamed<Int8Op, OUT, ADD, 2>(a, what, st);
    } else if (!fits) {
        // a whole row in one workgroup (262144 x 512 x 512: 150 us, through an fp32 row and quantize_rows 319)
        if (a.groups > kRowGroups) {
            LinearArgs b = a;
            b.pass = 1;
            if (int rc = launch_streamed<Int8Op, OUT, ADD, 2>(b, what, st)) return rc;
            b.pass = 2;
            return launch_streamed<Int8Op, OUT, ADD, 2>(b, what, st);
        }
        if (a.groups > 4) return launch_streamed<Int8Op, OUT, ADD, 4>(a, what, st);
        return launch_streamed<Int8Op, OUT, ADD, 2>(a, what, st);
    }
    if (nt == 4) return resident<OUT, 4, ADD>(a, what, st);
    if (nt == 2) return resident<OUT, 2, ADD>(a, what, st);
    return resident<OUT, 1, ADD>(a, what, st);
}

template <int OUT>
static int launch(const LinearArgs& a, int add_dtype, const char* what, hipStream_t st) {
    if (!a.addend) return launch<OUT, NO_ADD>(a, what, st);
    return add_dtype == NERF_F32 ? launch<OUT, NERF_F32>(a, what, st) : launch<OUT, NERF_BF16>(a, what, st);
}

// Checks and fields that both entry points share.
static int linear_args(LinearArgs& a, const char* what, const signed char* q, const float* scale, int64_t n, int k,
                       const void* packed, int m, const float* bias, const void* addend, int addend_dtype, int64_t ldadd, int relu) {
    if (int rc = require_widths(what, n, k, m)) return rc;
    NERF_REQUIRE(!addend || addend_dtype == NERF_F32 || addend_dtype == NERF_BF16, "%s: an addend is fp32 or bf16", what);
    if (n == 0) return 0;
    NERF_REQUIRE(q && scale && packed, "%s: null pointer", what);
    NERF_REQUIRE(!addend || ldadd >= m, "%s: rows of %d elements overlap", what, m);
    NERF_REQUIRE((((uintptr_t)q | (uintptr_t)packed) & 15) == 0 && (((uintptr_t)scale | (uintptr_t)bias) & 3) == 0 &&
                     (!addend || ((uintptr_t)addend & (dtype_size(addend_dtype) - 1)) == 0),
                 "%s: misaligned pointer", what);
    const PackedLayout lay(k, m, false);
    a.frags = (const char*)packed + lay.frags, a.groups = lay.mp / 64, a.steps = a.frag_steps = lay.kp / 64, a.n = n;
    a.q = q, a.scale = scale, a.features = m, a.wscale = (const float*)packed, a.bias = bias;
    a.addend = addend, a.ldadd = ldadd, a.relu = relu;
    return 0;
}

}  // namespace i8
}  // namespace nerf

using namespace nerf;
using namespace nerf::i8;

NERF_API int nerf_linear_int8(const signed char* q, const float* scale, int64_t n, int k, const void* packed, int m,
                              const float* bias, const void* addend, int addend_dtype, int64_t ldadd, int relu, void* y,
                              int dtype, int64_t ldy, nerf_stream_t stream) {
    const char* what = "nerf_linear_int8";
    LinearArgs a{};
    NERF_REQUIRE(dtype_ok(dtype), "%s: unknown type %d", what, dtype);
    if (int rc = linear_args(a, what, q, scale, n, k, packed, m, bias, addend, addend_dtype, ldadd, relu)) return rc;
    if (n == 0) return 0;
    NERF_REQUIRE(y && ldy >= m && ((uintptr_t)y & (dtype_size(dtype) - 1)) == 0, "%s: y must be aligned rows that do not overlap", what);
    a.out = y, a.ldout = ldy;
    hipStream_t st = as_stream(stream);
    if (dtype == NERF_F32) return launch<NERF_F32>(a, addend_dtype, what, st);
    if (dtype == NERF_F16) return launch<NERF_F16>(a, addend_dtype, what, st);
    return launch<NERF_BF16>(a, addend_dtype, what, st);
}

NERF_API size_t nerf_linear_int8_quantized_bytes(int64_t n, int m) {
    if (n < 1 || m < 1 || m > kMaxWidth) return 0;
    const int groups = (int)(up64(m) / 64);
    return groups > kRowGroups ? (size_t)n * ((groups + 3) / 4) * sizeof(unsigned) : 0;
}

NERF_API int nerf_linear_int8_quantized(const signed char* q, const float* scale, int64_t n, int k, const void* packed, int m,
                                        const float* bias, const void* addend, int addend_dtype, int64_t ldadd, int relu,
                                        int pow2, signed char* yq, float* yscale, unsigned char* ymask, void* workspace,
                                        size_t workspace_bytes, nerf_stream_t stream) {
    const char* what = "nerf_linear_int8_quantized";
    LinearArgs a{};
    if (int rc = linear_args(a, what, q, scale, n, k, packed, m, bias, addend, addend_dtype, ldadd, relu)) return rc;
    if (addend && m % 64 != 0)
        return NERF_FAIL(NERF_E_UNSUPPORTED, "%s: an addend of %d columns is not a whole number of 64", what, m);
    if (n == 0) return 0;
    NERF_REQUIRE(yq && yscale, "%s: null pointer", what);
    NERF_REQUIRE(((uintptr_t)yq & 15) == 0 && ((uintptr_t)yscale & 3) == 0 && ((uintptr_t)ymask & 1) == 0, "%s: misaligned pointer", what);
    const size_t need = nerf_linear_int8_quantized_bytes(n, m);
    NERF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 3) == 0),
                 "%s: needs a workspace of %zu bytes, got %zu", what, need, workspace ? workspace_bytes : 0);
    a.out = yq, a.out_scale = yscale, a.out_mask = ymask, a.tops = (unsigned*)workspace;
    hipStream_t st = as_stream(stream);
    if (pow2) return relu ? launch<TO_INT8 + 3>(a, addend_dtype, what, st) : launch<TO_INT8 + 2>(a, addend_dtype, what, st);
    return relu ? launch<TO_INT8 + 1>(a, addend_dtype, what, st) : launch<TO_INT8>(a, addend_dtype, what, st);
}
