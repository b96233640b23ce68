"""8-bit dense layers: every form of a call on every kernel that serves it."""
import pytest
import torch

from tests.test_int8_layers import TERMS, TYPES, close, dequantised, make

gpu_only = pytest.mark.gpu


# a row in one workgroup with its weights in LDS (one, two, three and four groups of channels), with streamed weights
# (to 256 channels, to 512), and in several workgroups
@gpu_only
@pytest.mark.parametrize("n,k,m", [(1, 1, 64), (33, 63, 64), (300, 128, 128), (500, 100, 192), (1000, 256, 256), (33000, 319, 256), (65, 500, 250),
                                   (13000, 640, 256), (12300, 1100, 200), (6000, 320, 512), (5200, 576, 320), (300, 64, 400), (12289, 700, 512),
                                   (9000, 256, 576), (7000, 700, 704), (4200, 64, 1024), (5000, 500, 1000)])
def test_8_bit_output_in_every_form(gpu, n, k, m):
    """With and without ReLU, scales that are powers of two, an addend of either type, and bits: those of the product
    stored in fp32 and quantised."""
    from nerf_amd import ops
    assert not ops._through_fp32(n, k, m)
    x, w, _, b = make(n, k, m, n + m, gpu)
    rows, packed = ops.quantize_rows(x - 0.3, pow2=True), ops.pack_int8(w, pow2=True)
    wide = torch.randn((n, m + 3), device=gpu)
    if n > 4:
        wide[n // 3, m // 2] = float("nan")
        wide[n - 2, 0] = float("inf")
    addends = (None, wide[:, :m], wide[:, 1:m + 1].bfloat16(), wide.bfloat16()[:, 3:]) if m % 64 == 0 else (None,)
    for relu in (False, True):
        for add in addends:
            for bias in (None, b):
                y = ops.linear_int8(rows, packed, bias, relu, add)
                for pow2 in (False, True):
                    want = ops.quantize_rows(y, pow2, True)
                    for mask in (False, True):
                        got = ops.linear_int8_quantized(rows, packed, bias, relu, add, pow2, mask)
                        assert torch.equal(got.q, want.q) and torch.equal(got.scale.nan_to_num(-1.), want.scale.nan_to_num(-1.)), (relu, pow2, mask)
                        assert torch.equal(got.mask, want.mask) if mask else got.mask is None, (relu, pow2)


@gpu_only
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("n,k", [(1, 1), (40, 64), (2500, 300), (33001, 27), (70001, 128), (9001, 1100)])
def test_weight_gradient_of_few_outputs(gpu, n, k, m, dtype):
    """Up to four outputs have a kernel of their own; one slice of the rows and many, one block of inputs and two, gradients
    that are contiguous and columns of a wider tensor."""
    from nerf_amd import ops
    t = TYPES[dtype]
    x, _, dz, _ = make(n, k, m + 2, 7 * n + m, gpu, t)
    rows = ops.quantize_rows(x, True)
    for d in (dz[:, :m].contiguous(), dz[:, 2:]):
        want, mag = dequantised(rows).t().contiguous() @ d.double(), dequantised(rows).abs().t().contiguous() @ d.double().abs()
        dw, db = ops.linear_int8_grad_weight(rows, d)
        # (a term of dz below 2^-126 may be taken as zero: 127 times that per row)
        close(dw, want, mag * TERMS[t] * n * 2.0 ** -23 + n * 2.0 ** -119, "dW")
        close(db, d.double().sum(0), d.double().abs().sum(0) * n * 2.0 ** -23 + 1e-38, "db")
        again = ops.linear_int8_grad_weight(rows, d)
        assert torch.equal(dw, again[0]) and torch.equal(db, again[1])


@gpu_only
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,k,m", [(40, 70, 96), (33000, 256, 256), (16500, 700, 704), (33000, 130, 33)])
def test_scales_that_are_not_powers_of_two_and_one_row_many_times(gpu, n, k, m, dtype):
    """The product takes rows and weights of different kinds of scales; rows that are the same give the same."""
    from nerf_amd import ops
    x, w, _, b = make(n, k, m, 3, gpu, TYPES[dtype])
    x[1:] = x[:1]
    for p2 in ((False, True), (True, False)):
        rows, packed = ops.quantize_rows(x, p2[0]), ops.pack_int8(w, p2[1])
        y = ops.linear_int8(rows, packed, b, dtype=TYPES[dtype])
        assert torch.equal(y, y[:1].expand(n, m))
        first = ops.quantize_rows(x[:1], p2[0])
        assert torch.equal(y[:1], ops.linear_int8(first, packed, b, dtype=TYPES[dtype]))
        q = ops.linear_int8_quantized(rows, packed, b, want_mask=True)
        r = ops.linear_int8_quantized(first, packed, b, want_mask=True)
        assert torch.equal(q.q, r.q.expand(n, -1)) and torch.equal(q.scale, r.scale.expand(n)) and torch.equal(q.mask, r.mask.expand(n, -1))
