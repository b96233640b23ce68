"""8-bit dense layers at the edges of their types: infinities, NaN, the largest and smallest numbers."""
import pytest
import torch

from tests.test_int8_layers import TERMS, TINY, TYPES, close, dequantised, make, ref_linear, unpack_bits

gpu_only = pytest.mark.gpu
# few rows (the direct kernel), weights in LDS, weights streamed; up to four outputs, 16-bit rows of odd width
KERNELS = [(40, 70, 96), (1500, 64, 3), (33000, 256, 256), (33000, 130, 33), (16500, 700, 704), (33001, 63, 4)]


def same_or_nan(got, want, bound, what):
    """Infinities of the same sign and NaN in the same places, everything else within the bound."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and bool(torch.isfinite(got[~inf & ~torch.isnan(want)]).all()), what
    fine = ~inf & ~torch.isnan(want)
    off = (got[fine] - want[fine]).abs() - bound[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()))


@gpu_only
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,k,m", KERNELS)
def test_an_infinite_gradient_is_infinite(gpu, n, k, m, dtype):
    """Products with an infinity are infinite, with zero NaN, as in the formula; no other row or column changes."""
    from nerf_amd import ops
    t = TYPES[dtype]
    x, w, dz, _ = make(n, k, m, 5, gpu, t)
    w[k // 2, :] = 0
    x[:, 0] = 1
    dz[n // 3, m // 2], dz[n - 1, 0] = float("inf"), -float("inf")
    rows, packed = ops.quantize_rows(x, True, True), ops.pack_int8(w, True)
    p, ws, _ = ref_linear(rows, w, True)
    wd, xd, d = p * ws, dequantised(rows), dz.double()
    far = torch.tensor([n // 3, n - 1], device=gpu)
    want = (d[far][:, None, :] * wd).sum(2)
    dx = ops.linear_int8_grad_input(dz, packed)
    same_or_nan(dx[far], want, torch.zeros_like(want), "dx")
    assert bool(torch.isinf(dx[far]).any()) and bool(torch.isnan(dx[far, k // 2]).all())
    rest = torch.ones(n, dtype=torch.bool, device=gpu)
    rest[far] = False
    clean = torch.where(torch.isinf(dz), torch.zeros_like(dz), dz)
    assert torch.equal(dx[rest], ops.linear_int8_grad_input(clean, packed)[rest])
    masked = ops.linear_int8_grad_input(dz, packed, rows.mask)
    on = unpack_bits(rows.mask, k)
    assert not bool(masked[~on].any()) and torch.equal(torch.nan_to_num(masked[on].float(), 7, 8, 9), torch.nan_to_num(dx[on].float(), 7, 8, 9))
    dw, db = ops.linear_int8_grad_weight(rows, dz)
    for j in {0, m // 2}:
        same_or_nan(dw[:, j], (xd * d[:, j:j + 1]).sum(0), torch.full((k,), float("inf"), dtype=torch.float64, device=gpu), "dW")
        assert bool(torch.isinf(db[j]))
    keep = [j for j in range(m) if j not in (0, m // 2)]
    dwc, dbc = ops.linear_int8_grad_weight(rows, clean)
    assert torch.equal(dw[:, keep], dwc[:, keep]) and torch.equal(db[keep], dbc[keep])


@gpu_only
@pytest.mark.parametrize("n,k,m", KERNELS)
def test_gradients_of_the_largest_and_smallest_size(gpu, n, k, m):
    """fp32 gradients up to the largest float, and down to 2^-126, whose products are ordinary numbers."""
    from nerf_amd import ops
    big = torch.finfo(torch.float32).max
    x, w, dz, _ = make(n, k, m, 6, gpu)
    g = torch.Generator(device=gpu).manual_seed(8)
    # within half a bf16 step of the largest float and elsewhere in its last binade
    dz = big * (1 - torch.rand((n, m), generator=g, device=gpu) * 0.5) * (torch.rand((n, m), generator=g, device=gpu) - 0.5).sign()
    dz[::2] = big
    for scale, name in ((1.0, "large"), (2.0 ** -250, "small")):
        d32 = (dz.double() * scale).float()
        up = 2.0 ** -60 if scale == 1.0 else 2.0 ** 60
        rows, packed = ops.quantize_rows(x * up, True, True), ops.pack_int8(w * up, True)
        p, ws, _ = ref_linear(rows, w * up, True)
        wd, xd, d = p * ws, dequantised(rows), d32.double()
        # (a bf16 term below 2^-126 may be taken as zero: at most 2^-126 of it, times the other factor)
        lost = 2.0 ** -125
        want, mag = d @ wd.t().contiguous(), d.abs() @ wd.abs().t().contiguous()
        close(ops.linear_int8_grad_input(d32, packed), want, mag * (3 * m * 2.0 ** -23 + 2.0 ** -24) + lost * wd.abs().sum(1) + 1e-38, name + " dx")
        dw, _ = ops.linear_int8_grad_weight(rows, d32)
        close(dw, xd.t().contiguous() @ d, xd.abs().t().contiguous() @ d.abs() * 3 * n * 2.0 ** -23 + lost * xd.abs().sum(0)[:, None] + 1e-38, name + " dW")


@gpu_only
@pytest.mark.parametrize("n,k,m", [(40, 70, 96), (33000, 256, 192), (16500, 700, 704), (16500, 512, 512), (9000, 256, 576)])
def test_a_nan_of_either_sign_passes_a_relu(gpu, n, k, m):
    """A row's scale, a bias, an addend that is NaN with its sign bit set, and the difference of two infinities."""
    from nerf_amd import ops
    x, w, _, b = make(n, k, m, 7, gpu)
    rows, packed = ops.quantize_rows(x.abs() + 0.1), ops.pack_int8(w)
    neg = torch.tensor([-1], dtype=torch.int32, device=gpu).view(torch.float32)
    at = [0, n // 2, n - 1]

    def check(y, q, where, col=slice(None)):
        assert bool(torch.isnan(y[where, col]).all())
        assert bool(torch.isnan(q.scale[where]).all()) and not bool(q.q[where].any())
    scale = rows.scale.clone()
    scale[at] = neg
    bad = ops.Int8Rows(rows.q, scale, k)
    bias = b.clone()
    bias[m // 2] = neg[0]
    add = torch.zeros((n, m), device=gpu)
    add[at] = neg
    both = lambda *a, **kw: (ops.linear_int8(*a, relu=True, **kw), ops.linear_int8_quantized(*a, relu=True, want_mask=True, **kw))
    check(*both(bad, packed, b), at)
    check(*both(rows, packed, bias), slice(None), m // 2)
    check(*both(rows, packed, b, addend=add), at)
    # sums of either sign times an infinite scale, plus the other infinity
    inf = float("inf")
    scale[at] = inf
    sums = ops.linear_int8(ops.Int8Rows(rows.q, torch.ones_like(scale), k), packed)[0]
    opposite = torch.where(sums > 0, torch.full_like(b, -inf), torch.full_like(b, inf))
    y, q = both(ops.Int8Rows(rows.q, scale, k), packed, opposite)
    check(y[:1], q, slice(0, 1))
    want = torch.relu(opposite)
    assert torch.equal(y[1], want)                           # a finite row plus an infinite bias


@pytest.mark.parametrize("n,k,m,two", [(2048, 640, 64, True), (16384, 640, 64, False), (8192, 896, 128, True), (8192, 640, 256, True), (12288, 640, 256, False),
                                       (4096, 640, 512, True), (8192, 640, 512, False), (100, 576, 256, False), (1, 64, 512, False),
                                       (4096, 256, 576, True), (8192, 256, 576, False), (2048, 512, 2048, True), (4096, 512, 2048, False),
                                       (32768, 640, 1024, False), (32768, 1024, 1024, True), (131072, 1024, 1024, False), (32768, 2048, 2048, True), (162501, 120, 1271, False)])
def test_an_8_bit_output_takes_the_way_that_was_measured_faster(n, k, m, two):
    from nerf_amd import ops
    assert ops._through_fp32(n, k, m) is two
