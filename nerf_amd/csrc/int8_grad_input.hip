// nerf_linear_int8_grad_input: dz times the transposed weights, which are exact in bf16.
#include "int8_product.h"

namespace nerf {
namespace i8 {

// Steps of dz rows in a unit: 256 columns of 16-bit types, 128 of fp32 (32 registers).
template <int DT> constexpr int kHeld = DT == NERF_F32 ? 4 : 8;

template <int DT, int NT>
static int resident(const LinearArgs& a, const char* what, hipStream_t st) {
    if (a.width % 32 != 0) return launch_resident<Bf16Op<DT, false>, DT, NT, 2, 1, NO_ADD>(a, what, st);
    if (a.steps <= 2) return launch_resident<Bf16Op<DT, true>, DT, NT, 2, 1, NO_ADD>(a, what, st);
    return launch_resident<Bf16Op<DT, true>, DT, NT, kHeld<DT>, 1, NO_ADD>(a, what, st);
}

template <int DT>
static int launch(const LinearArgs& a, const char* what, hipStream_t st) {
    const int nt = resident_groups(a);
    // (fp16 and fp32 rows cannot go to LDS as they are: their terms are formed in registers)
    const bool streamed = DT == NERF_BF16 && (nt == 0 || a.groups > nt) && a.width % 32 == 0 && a.lddz % 8 == 0 && ((uintptr_t)a.dz & 15) == 0;
    if (few_rows(a, streamed) || (nt == 0 && !streamed)) return launch_direct<Bf16Op<DT, false>, DT, NO_ADD>(a, what, st);
    if constexpr (DT == NERF_BF16) {
        if (streamed) return launch_streamed<Bf16Op<DT, true>, DT, NO_ADD, 2>(a, what, st);
    }
    if (nt == 4) return resident<DT, 4>(a, what, st);
    if (nt == 3) return resident<DT, 3>(a, what, st);
    if (nt == 2) return resident<DT, 2>(a, what, st);
    return resident<DT, 1>(a, what, st);
}

}  // namespace i8
}  // namespace nerf

using namespace nerf;
using namespace nerf::i8;

NERF_API int nerf_linear_int8_grad_input(const void* dz, int dtype, int64_t n, int m, int64_t lddz, const void* packed,
                                         int k, const unsigned char* mask, void* dx, int64_t lddx, nerf_stream_t stream) {
    const char* what = "nerf_linear_int8_grad_input";
    if (int rc = require_widths(what, n, k, m)) return rc;
    NERF_REQUIRE(dtype_ok(dtype), "%s: unknown type %d", what, dtype);
    if (n == 0) return 0;
    NERF_REQUIRE(dz && packed && dx, "%s: null pointer", what);
    NERF_REQUIRE(lddz >= m && lddx >= k, "%s: rows overlap", what);
    NERF_REQUIRE(((uintptr_t)packed & 15) == 0 && (((uintptr_t)dz | (uintptr_t)dx) & (dtype_size(dtype) - 1)) == 0 &&
                     ((uintptr_t)mask & 7) == 0,
                 "%s: misaligned pointer", what);
    const PackedLayout lay(k, m, true);
    LinearArgs a{};
    a.frags = (const char*)packed + lay.frags_t, a.groups = lay.kp / 64, a.steps = (m + 31) / 32, a.frag_steps = lay.mp / 32, a.n = n;
    a.dz = dz, a.lddz = lddz, a.width = m, a.features = k, a.mask = mask, a.out = dx, a.ldout = lddx;
    hipStream_t st = as_stream(stream);
    if (dtype == NERF_F32) return launch<NERF_F32>(a, what, st);
    if (dtype == NERF_F16) return launch<NERF_F16>(a, what, st);
    return launch<NERF_BF16>(a, what, st);
}
