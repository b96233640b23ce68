"""Dense layers in 8 bits: rows and weights in integers, the product, its two gradients.

Plain implementations in 64 bits.  Tolerances: a rounding to a type is off by at most finfo(t).eps / 2 of
the value; a sum of c terms in fp32 by at most c 2^-23 of the sum of their magnitudes, whatever the order
(2^-23: a matrix instruction may truncate)."""
import ctypes

import numpy as np
import pytest
import torch

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
TERMS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}   # bf16 terms of an element of dz
TINY = {t: max(torch.finfo(t).smallest_normal * torch.finfo(t).eps, 1e-38) for t in TERMS}   # below the normal numbers: a step
SHAPES = [(1, 1, 1), (1, 256, 256), (3, 63, 5), (17, 64, 64), (31, 65, 63), (33, 128, 3), (64, 319, 256), (257, 283, 128),
          (1000, 27, 129), (130, 2048, 17), (65, 130, 700), (4100, 256, 256), (129, 600, 1), (16, 2047, 33),
          (4111, 63, 256), (4099, 283, 128), (5003, 319, 256), (4097, 128, 3), (6001, 27, 70), (4133, 700, 200), (4100, 1100, 65), (33000, 256, 192), (70001, 64, 64), (5000, 100, 96), (4200, 640, 600), (4500, 576, 1000), (4300, 1000, 576), (6000, 512, 512), (4200, 832, 190), (4100, 640, 150),
          (300, 1000, 320), (5000, 40, 400), (9000, 100, 510), (1, 2, 300), (700, 200, 1344), (1, 65, 513), (70001, 1024, 512), (524817, 250, 200),
          (32801, 63, 256), (32771, 283, 128), (32800, 319, 256), (32770, 128, 3), (33001, 27, 70), (32777, 100, 96), (32773, 832, 190),
          (32800, 640, 150), (32769, 1, 1), (40001, 576, 130), (4111, 1100, 1100), (9000, 700, 704), (16500, 512, 512), (16501, 96, 576)]


# ---- without a GPU -----------------------------------------------------------------------------------
def test_bad_arguments_are_refused_without_a_gpu():
    from nerf_amd import _native
    lib = _native.lib()
    one = ctypes.c_void_p(4096)      # never read: every call below is refused
    odd = ctypes.c_void_p(4097)
    assert lib.nerf_quantize_rows(None, 0, 4, 8, 8, 0, None, None, None, None) == -1
    assert b"nerf_quantize_rows" in lib.nerf_last_error()
    assert lib.nerf_quantize_rows(one, 0, -1, 8, 8, 0, one, one, None, None) == -1
    assert lib.nerf_quantize_rows(one, 0, 4, 0, 8, 0, one, one, None, None) == -1
    assert lib.nerf_quantize_rows(one, 0, 4, 65537, 65537, 0, one, one, None, None) == -1
    assert lib.nerf_quantize_rows(one, 3, 4, 8, 8, 0, one, one, None, None) == -1
    assert lib.nerf_quantize_rows(one, 0, 4, 8, 7, 0, one, one, None, None) == -1
    assert lib.nerf_quantize_rows(odd, 0, 4, 8, 8, 0, one, one, None, None) == -1
    assert lib.nerf_quantize_rows(one, 0, 4, 8, 8, 0, odd, one, None, None) == -1
    assert lib.nerf_quantize_rows(None, 0, 0, 8, 8, 0, None, None, None, None) == 0     # no rows: nothing to do
    assert lib.nerf_int8_packed_bytes(0, 4, 0) == 0 and lib.nerf_int8_packed_bytes(4, 65537, 0) == 0
    assert lib.nerf_int8_packed_bytes(63, 65, 0) == 128 * 4 + 128 * 64
    assert lib.nerf_int8_packed_bytes(63, 65, 1) == 128 * 4 + 128 * 64 * 3
    assert lib.nerf_int8_pack(None, 4, 4, 0, one, None) == -1
    assert lib.nerf_int8_pack(one, 4, 4, 0, odd, None) == -1
    assert lib.nerf_int8_pack(one, 65537, 4, 0, one, None) == -1
    linear = lambda **c: lib.nerf_linear_int8(*[{**dict(q=one, scale=one, n=4, k=8, packed=one, m=8, bias=None, addend=None, adt=0,
                                                        ldadd=0, relu=0, y=one, dt=0, ldy=8, st=None), **c}[x] for x in
                                                ("q", "scale", "n", "k", "packed", "m", "bias", "addend", "adt", "ldadd", "relu", "y", "dt", "ldy", "st")])
    for bad in (dict(q=None), dict(q=odd), dict(packed=None), dict(y=None), dict(scale=None), dict(k=0), dict(m=0), dict(n=-1), dict(m=70000),
                dict(dt=5), dict(ldy=7), dict(addend=one, ldadd=7), dict(addend=one, ldadd=8, adt=9), dict(bias=odd), dict(y=odd)):
        assert linear(**bad) == -1, bad
    assert linear(n=0, q=None) == 0
    size = lib.nerf_linear_int8_quantized_bytes
    assert size(10, 512) == 0 and size(10, 513) == 10 * 3 * 4 and size(1, 65536) == 256 * 4 and size(0, 600) == 0 and size(5, 65537) == 0
    quant = lambda **c: lib.nerf_linear_int8_quantized(*[{**dict(q=one, scale=one, n=4, k=8, packed=one, m=8, bias=None, addend=None, adt=0, ldadd=0,
                                                                 relu=0, pow2=0, yq=one, ys=one, ym=None, ws=None, size=0, st=None), **c}[x] for x in
                                                         ("q", "scale", "n", "k", "packed", "m", "bias", "addend", "adt", "ldadd", "relu", "pow2", "yq", "ys", "ym", "ws", "size", "st")])
    for bad in (dict(q=None), dict(yq=None), dict(ys=None), dict(yq=odd), dict(ym=odd), dict(k=0), dict(m=0), dict(n=-1), dict(addend=one, ldadd=7), dict(m=513), dict(m=513, ws=one, size=47),
                dict(m=513, ws=odd, size=48)):
        assert quant(**bad) == -1, bad
    assert quant(m=65, addend=one, ldadd=65) == -2
    assert quant(m=64, addend=one, ldadd=64, adt=1) == -1      # an addend is fp32 or bf16
    gi = lambda **c: lib.nerf_linear_int8_grad_input(*[{**dict(dz=one, dt=0, n=4, m=8, lddz=8, packed=one, k=8, mask=None, dx=one, lddx=8, st=None), **c}[x]
                                                       for x in ("dz", "dt", "n", "m", "lddz", "packed", "k", "mask", "dx", "lddx", "st")])
    for bad in (dict(dz=None), dict(dx=None), dict(packed=odd), dict(dt=3), dict(lddz=7), dict(lddx=7), dict(mask=odd), dict(k=0), dict(n=-1)):
        assert gi(**bad) == -1, bad
    need = lib.nerf_linear_int8_grad_weight_bytes(4096, 64, 64)
    assert need == 16 * 65 * 64 * 4 and lib.nerf_linear_int8_grad_weight_bytes(4, 64, 64) == 0
    gw = lambda **c: lib.nerf_linear_int8_grad_weight(*[{**dict(q=one, scale=one, n=4096, k=64, dz=one, dt=0, m=64, lddz=64, dw=one, db=one, ws=one, nb=need, st=None), **c}[x]
                                                        for x in ("q", "scale", "n", "k", "dz", "dt", "m", "lddz", "dw", "db", "ws", "nb", "st")])
    for bad in (dict(q=None), dict(dz=None), dict(dw=None), dict(db=None), dict(n=0), dict(m=0), dict(dt=7), dict(lddz=63), dict(ws=None), dict(nb=need - 1), dict(q=odd)):
        assert gw(**bad) == -1, bad
    assert b"workspace" in (gw(nb=0), lib.nerf_last_error())[1]


def test_no_cpu_fallback():
    from nerf_amd import _native, ops
    x = torch.zeros((4, 8))
    for call in (lambda: ops.quantize_rows(x), lambda: ops.pack_int8(x), lambda: ops.Int8Rows(torch.zeros((4, 64), dtype=torch.int8), torch.zeros(4), 8)):
        with pytest.raises(_native.NerfHipError):
            call()


def test_packed_weights_of_another_size_are_refused():
    from nerf_amd import _native, ops
    need = _native.lib().nerf_int8_packed_bytes(70, 5, 1)
    assert ops.Int8Weights(torch.zeros(need, dtype=torch.uint8), 70, 5, True).m == 5
    for packed, k, m, pow2 in ((torch.zeros(need - 1, dtype=torch.uint8), 70, 5, True), (torch.zeros(need, dtype=torch.uint8), 70, 5, False),
                               (torch.zeros(need, dtype=torch.int8), 70, 5, True), (torch.zeros(2 * need, dtype=torch.uint8)[::2], 70, 5, True),
                               (torch.zeros(0, dtype=torch.uint8), 0, 5, True)):
        with pytest.raises(ValueError):
            ops.Int8Weights(packed, k, m, pow2)


# ---- plain forms ---------------------------------------------------------------------------------------
def ref_scale(top, pow2):
    """Scales of float32 magnitudes, in float64."""
    top = top.double()
    if pow2:
        _, e = torch.frexp(top / 127.0 * (1 - 2.0 ** -40))          # smallest power of two >= top / 127
        e = torch.where(top > 0, e, torch.full_like(e, -200)).clamp_min(-126)
        return ((e.long() + 1023) << 52).view(torch.float64)
    return torch.where(top < 2.0 ** -100, torch.zeros_like(top), top / 127.0)


def dequantised(rows):
    return rows.q[:, :rows.k].double() * rows.scale.double()[:, None]


def unpack_bits(mask, k):
    return ((mask[:, :, None] >> torch.arange(8, device=mask.device, dtype=torch.uint8)) & 1).reshape(mask.shape[0], -1)[:, :k].bool()


def make(n, k, m, seed, gpu, dtype=torch.float32):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.relu(torch.randn((n, k), generator=g, device=gpu)) * torch.exp(torch.randn((n, 1), generator=g, device=gpu))
    if n > 1:
        x[n // 2] = 0                                                   # a row that is empty
    w = torch.randn((k, m), generator=g, device=gpu) / k ** 0.5
    w[:, m // 2] *= 1e-3
    dz = torch.randn((n, m), generator=g, device=gpu) * 10.0 ** (-4 * torch.rand((n, 1), generator=g, device=gpu))
    b = torch.randn((m,), generator=g, device=gpu)
    return x.to(dtype), w, dz.to(dtype), b


def close(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs() - bound
    assert not bool(torch.isnan(got).any()) and float(off.max()) <= 0, f"{what}: {float(off.max()):.3g} beyond the bound"


def inverse127(top):
    """127 / top with one rounding (a python number divided by a tensor is its reciprocal times the number: two)."""
    return torch.from_numpy(np.float32(127) / top.cpu().numpy()).to(top.device)


gpu_only = pytest.mark.gpu


# ---- quantised rows -------------------------------------------------------------------------------------
@gpu_only
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,k", [(1, 1), (5, 3), (64, 256), (33, 63), (7, 512), (9, 513), (4, 1000), (3, 2048), (2, 2049), (3, 5000), (2, 65536), (3001, 319)])
def test_quantize_rows(gpu, n, k, dtype, pow2):
    from nerf_amd import ops
    x = make(n, k, 1, n + k, gpu, TYPES[dtype])[0] - 0.25
    x[0, 0] = -x.abs().max() * 1.5 - 1
    rows = ops.quantize_rows(x, pow2=pow2, want_mask=True)
    assert rows.q.shape == (n, -(-k // 64) * 64) and not bool(rows.q[:, k:].any())
    xf = x.float()
    top = xf.abs().amax(1)
    want = ref_scale(top, pow2)
    assert float(((rows.scale.double() - want).abs() - 2.0 ** -24 * want).max()) <= 0      # one rounding (none for a power of two)
    if pow2:
        assert torch.equal(rows.scale.double(), want)
    # half a step, and the roundings of the scale's inverse, of the product and of the scale: 3 x 2^-24 of 127 steps
    err = (dequantised(rows) - xf.double()).abs()
    assert float((err - (0.5 + (0 if pow2 else 127 * 3 * 2.0 ** -24)) * rows.scale.double()[:, None]).max()) <= 0
    assert int(rows.q.int().abs().max()) <= 127
    assert torch.equal(unpack_bits(rows.mask, k), x > 0) and not bool(unpack_bits(rows.mask, rows.q.shape[1])[:, k:].any())
    # the integers by the formula, bit for bit
    inv = (1 / rows.scale) if pow2 else inverse127(top)
    assert torch.equal(rows.q[:, :k].float(), torch.round(xf * inv[:, None]))


@gpu_only
@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_rows_special_values(gpu, pow2):
    from nerf_amd import ops
    inf, nan = float("inf"), float("nan")
    x = torch.zeros((12, 70), device=gpu)
    x[1, 3] = 1e-44                      # a subnormal
    x[2, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])   # halves go to the even integer
    x[3, 69] = 3.4e38
    x[4, 2], x[4, 3] = inf, 1.0
    x[5, 68], x[5, 3] = nan, 1.0
    x[6, 0] = -inf
    x[7, :2] = torch.tensor([-0.0, 2.0 ** -101])
    x[8, :2] = torch.tensor([2.0 ** -100, -(2.0 ** -101)])
    x[9] = 127.0
    x[10, 1] = 127.00001
    x[11, 0] = torch.finfo(torch.float32).tiny
    rows = ops.quantize_rows(x, pow2=pow2, want_mask=True)
    q, s = rows.q.cpu(), rows.scale.cpu()
    for r in (4, 5, 6):
        assert bool(torch.isnan(s[r])) and not bool(q[r].any())
    assert torch.equal(unpack_bits(rows.mask, 70), x > 0)                # NaN is not positive, infinity is
    assert not bool(q[0].any()) and float(s[0]) == (2.0 ** -126 if pow2 else 0.0)
    assert q[2, :4].tolist() == [127, 0, 2, -2] and float(s[2]) == 1.0
    assert (q[9, :70] == 127).all() and float(s[9]) == 1.0
    fine = [0, 1, 2, 3, 7, 8, 9, 10, 11]
    assert bool(torch.isfinite(s[fine]).all())
    if pow2:
        assert float(s[10]) == 2.0 and int(q[10, 1]) == 64
        assert float(s[3]) == 2.0 ** 122 and float(s[1]) == 2.0 ** -126 and float(s[7]) == 2.0 ** -107
    else:
        assert not bool(q[7].any()) and float(s[7]) == 0.0 and not bool(q[1].any()) and not bool(q[11].any())
        assert int(q[3, 69]) == 127 and int(q[8, 0]) == 127 and int(q[8, 1]) == -64      # -63.5: to the even one


@gpu_only
@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides_and_alignment(gpu, dtype):
    """Rows that start at odd addresses, rows of a wider tensor, transposed and broadcast ones."""
    from nerf_amd import ops
    t = TYPES[dtype]
    n, k, m = 37, 75, 19
    base, w, dz, _ = make(n, k + 9, m + 6, 5, gpu, t)
    w = w[:k, :m].contiguous()
    packed = ops.pack_int8(w, pow2=True)
    for x in (base[:, :k], base[:, 1:k + 1], base[:, 3:k + 3], base[:, :k].t().contiguous().t(), base[:1, :k].expand(n, k), base[::2, 5:k + 5]):
        a, b = ops.quantize_rows(x, True, True), ops.quantize_rows(x.clone(memory_format=torch.contiguous_format), True, True)
        assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale) and torch.equal(a.mask, b.mask)
    rows = ops.quantize_rows(base[:, :k], True, True)
    for d in (dz[:, :m], dz[:, 1:m + 1], dz[:, 5:m + 5], dz[:, :m].t().contiguous().t(), dz[:1, :m].expand(n, m)):
        c = d.clone(memory_format=torch.contiguous_format)
        assert torch.equal(ops.linear_int8_grad_input(d, packed, rows.mask), ops.linear_int8_grad_input(c, packed, rows.mask))
        for u, v in zip(ops.linear_int8_grad_weight(rows, d), ops.linear_int8_grad_weight(rows, c)):
            assert torch.equal(u, v)
        assert torch.equal(ops.linear_int8(rows, packed, addend=d), ops.linear_int8(rows, packed, addend=c))
    assert torch.equal(ops.pack_int8(w.t().contiguous().t(), True).packed, packed.packed)


# ---- the product -------------------------------------------------------------------------------------------
def ref_linear(rows, w, pow2):
    """(integers of W, channel scales, exact sums), all in 64 bits."""
    top = w.abs().amax(0)
    s = ref_scale(top, pow2)
    s32 = s.float()
    inv = (1 / s32) if pow2 else torch.where(s32 > 0, inverse127(top), torch.zeros_like(s32))
    p = torch.round(w * inv[None, :]).double()
    return p, s32.double(), rows.q[:, :rows.k].double() @ p             # |sum| < 2^31: exact


@gpu_only
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,k,m", SHAPES)
def test_linear_int8(gpu, n, k, m, dtype, pow2):
    from nerf_amd import ops
    t = TYPES[dtype]
    x, w, _, b = make(n, k, m, n + k + m, gpu)
    rows, packed = ops.quantize_rows(x, pow2=pow2), ops.pack_int8(w, pow2=pow2)
    p, ws, sums = ref_linear(rows, w, pow2)
    prod = sums * ws * rows.scale.double()[:, None]
    half = torch.finfo(t).eps / 2
    for bias, add, relu in ((None, None, False), (b, None, True), (b, torch.randn((n, m), device=gpu).to(t), False), (None, torch.randn((n, m), device=gpu), True)):
        want = prod + (0 if bias is None else bias.double()) + (0 if add is None else add.double())
        mag = prod.abs() + (0 if bias is None else bias.double().abs()) + (0 if add is None else add.double().abs())
        want = want.clamp(min=0) if relu else want
        got = ops.linear_int8(rows, packed, bias, relu=relu, addend=add, dtype=t)
        assert got.dtype == t
        # sum, two scales, bias and addend: five roundings of 2^-24, each of at most `mag` (1 + 2^-22); then the type's
        close(got, want, mag * 5.001 * 2.0 ** -24 + half * (want.abs() + mag * 2.0 ** -20) + TINY[t], (n, k, m, dtype))
    # by the formula in fp32: the sum and its product with the channel scale are rounded, then the product with
    # the row scale plus the bias once (exact in 64 bits but for a last rounding there, which can move the
    # one to fp32 by a step when it falls on a tie: never for power-of-two scales here)
    y64 = (sums.float() * ws.float()).double() * rows.scale.double()[:, None] + b.double()
    y = ops.linear_int8(rows, packed, b)
    assert float((y.double() - y64).abs().sub(2.0 ** -24 * (1 + 2.0 ** -20) * y64.abs()).max()) <= 1e-40
    if pow2:
        assert torch.equal(y, (sums.float() * ws.float()) * rows.scale[:, None] + b)
    # and in 8 bits again: as if y had been stored in fp32 and quantised
    y = torch.relu(y)
    for p2 in (False, True):
        a, c = ops.linear_int8_quantized(rows, packed, b, relu=True, pow2=p2, want_mask=True), ops.quantize_rows(y, p2, True)
        assert a.k == m and a.pow2 == p2
        assert torch.equal(a.q, c.q) and torch.equal(a.scale, c.scale) and torch.equal(a.mask, c.mask)
    a = ops.linear_int8_quantized(rows, packed, addend=y)
    c = ops.quantize_rows(ops.linear_int8(rows, packed, addend=y))
    assert torch.equal(a.q, c.q) and torch.equal(a.scale, c.scale) and a.mask is None


@gpu_only
def test_linear_int8_extremes(gpu):
    """The largest sums, a row and a channel that are not finite, and sums beyond 24 bits."""
    from nerf_amd import ops
    k = 65536
    rows = ops.Int8Rows(torch.full((2, k), 127, dtype=torch.int8, device=gpu), torch.ones(2, device=gpu), k)
    w = torch.full((k, 2), 127.0, device=gpu)
    w[:, 1] = -127.0
    y = ops.linear_int8(rows, ops.pack_int8(w))
    assert torch.equal(y, torch.tensor([[1.0, -1.0]] * 2, device=gpu) * float(np.float32(127 * 127 * k)))
    x = torch.randn((40, 33), device=gpu)
    x[3, 7], x[20, 0] = float("nan"), float("inf")
    w = torch.randn((33, 5), device=gpu)
    w[2, 4] = float("inf")
    good = ops.linear_int8(ops.quantize_rows(x[:3]), ops.pack_int8(w[:, :4].contiguous()), relu=True)
    rows = ops.quantize_rows(x, pow2=True, want_mask=True)
    y = ops.linear_int8(ops.quantize_rows(x), ops.pack_int8(w), relu=True)
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[20]).all()) and bool(torch.isnan(y[:, 4]).all())
    assert torch.equal(y[:3, :4], good)
    q = ops.linear_int8_quantized(ops.quantize_rows(x), ops.pack_int8(w[:, :4].contiguous()), relu=True, want_mask=True)
    assert bool(torch.isnan(q.scale[[3, 20]]).all()) and not bool(q.q[[3, 20]].any()) and not bool(q.mask[[3, 20]].any())
    assert bool(torch.isfinite(q.scale[:3]).all())
    dx = ops.linear_int8_grad_input(torch.ones((40, 5), device=gpu), ops.pack_int8(w, True), rows.mask)
    on = unpack_bits(rows.mask, 33)
    assert bool(torch.isnan(dx[on]).all()) and not bool(dx[~on].any())
    dw, db = ops.linear_int8_grad_weight(rows, torch.ones((40, 5), device=gpu))
    assert bool(torch.isnan(dw).all()) and torch.equal(db, torch.full((5,), 40.0, device=gpu))


# ---- the gradients -------------------------------------------------------------------------------------------
@gpu_only
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,k,m", SHAPES)
def test_gradients(gpu, n, k, m, dtype):
    from nerf_amd import ops
    t = TYPES[dtype]
    x, w, dz, _ = make(n, k, m, 3 * n + k + m, gpu, t)
    rows, packed = ops.quantize_rows(x, True, True), ops.pack_int8(w, True)
    p, ws, _ = ref_linear(rows, w, True)
    wd, xd, d = p * ws, dequantised(rows), dz.double()
    want, mag = d @ wd.t().contiguous(), d.abs() @ wd.abs().t().contiguous()
    bound = mag * TERMS[t] * m * 2.0 ** -23 + torch.finfo(t).eps / 2 * want.abs() + TINY[t]
    close(ops.linear_int8_grad_input(dz, packed), want, bound * 1.01, "dx")
    on = unpack_bits(rows.mask, k)
    dx = ops.linear_int8_grad_input(dz, packed, rows.mask)
    close(dx, want * on, bound * on * 1.01, "masked dx")
    dw, db = ops.linear_int8_grad_weight(rows, dz)
    # (a term of dz below 2^-126, bf16's smallest normal number, may be taken as zero: 127 times that per row)
    close(dw, xd.t().contiguous() @ d, xd.abs().t().contiguous() @ d.abs() * TERMS[t] * n * 2.0 ** -23 + n * 2.0 ** -119, "dW")
    close(db, d.sum(0), d.abs().sum(0) * n * 2.0 ** -23 + 1e-38, "db")
    again = ops.linear_int8_grad_weight(rows, dz)
    assert torch.equal(dw, again[0]) and torch.equal(db, again[1])


@gpu_only
def test_gradients_against_differences(gpu):
    """sum(g relu(x^ W^ + b)) moved along a bias, an integer of W^ and an integer of x^: with power-of-two
    scales the function is piecewise linear in each and the steps below are exact in fp32 up to the sums'
    roundings, which 1e-4 of the gradients' size covers (24 terms of 2^-24, steps of 2^-7)."""
    from nerf_amd import ops
    n, k, m = 6, 12, 4
    x, w, _, b = make(n, k, m, 11, gpu)
    x = x + 0.5
    g = torch.randn((n, m), device=gpu)
    rows, packed = ops.quantize_rows(x, True, True), ops.pack_int8(w, True)
    y = ops.linear_int8(rows, packed, b, relu=True)
    dz = g * (y > 0)
    dx = ops.linear_int8_grad_input(dz, packed)
    dw, db = ops.linear_int8_grad_weight(rows, dz)
    xd = dequantised(rows)
    p, ws, _ = ref_linear(rows, w, True)
    wd = p * ws
    f = lambda xx, ww, bb: float((g.double() * (xx @ ww + bb).clamp(min=0)).sum())
    z = xd @ wd + b.double()
    h = float(z.abs().min()) * 1e-3 / (1 + float(xd.abs().max() + wd.abs().max()))    # no unit changes sides
    for got, i, which in [(dx, (2, 5), 0), (dx, (0, 0), 0), (dw, (3, 1), 1), (dw, (11, 3), 1), (db, (2,), 2)]:
        args = [xd.clone(), wd.clone(), b.double().clone()]
        args[which][i] += h
        up = f(*args)
        args[which][i] -= 2 * h
        assert abs((up - f(*args)) / (2 * h) - float(got[i])) <= 1e-4 * (1 + abs(float(got[i])))


# ---- refusals, empty calls, streams, graphs -----------------------------------------------------------------------
@gpu_only
def test_refusals(gpu):
    from nerf_amd import _native, ops
    x, w, dz, b = make(8, 10, 6, 1, gpu)
    rows, packed = ops.quantize_rows(x), ops.pack_int8(w)
    rows2, packed2 = ops.quantize_rows(x, True, True), ops.pack_int8(w, True)
    bad = [lambda: ops.quantize_rows(x.double()), lambda: ops.quantize_rows(x[0]), lambda: ops.quantize_rows(x[:, :0]),
           lambda: ops.pack_int8(w[0]), lambda: ops.pack_int8(w[:0]), lambda: ops.pack_int8(torch.zeros((1, 65537), device=gpu)),
           lambda: ops.Int8Rows(rows.q[:, :10], rows.scale, 10), lambda: ops.Int8Rows(rows.q, rows.scale[:3], 10), lambda: ops.Int8Rows(rows.q, rows.scale, 65),
           lambda: ops.Int8Rows(rows.q.short(), rows.scale, 10), lambda: ops.Int8Rows(rows.q, rows.scale.double(), 10),
           lambda: ops.Int8Rows(rows.q, rows.scale, 10, mask=rows2.mask[:4]), lambda: ops.Int8Rows(rows.q, torch.zeros((16,), device=gpu)[::2], 10),
           lambda: ops.linear_int8(x, packed), lambda: ops.linear_int8(rows, w), lambda: ops.linear_int8(ops.quantize_rows(x[:, :9]), packed),
           lambda: ops.linear_int8(rows, packed, b[:5]), lambda: ops.linear_int8(rows, packed, dtype=torch.int8), lambda: ops.linear_int8(rows, packed, addend=dz[:7]),
           lambda: ops.linear_int8(rows, packed, addend=x), lambda: ops.linear_int8_grad_input(dz, packed), lambda: ops.linear_int8_grad_input(dz[:, :5], packed2),
           lambda: ops.linear_int8_grad_input(dz, packed2, rows2.mask[:3]), lambda: ops.linear_int8_grad_input(dz, packed2, rows2.mask.int()),
           lambda: ops.linear_int8_grad_input(dz.long(), packed2), lambda: ops.linear_int8_grad_weight(rows, dz), lambda: ops.linear_int8_grad_weight(rows2, dz[:7]),
           lambda: ops.linear_int8_grad_weight(rows2, dz[0]), lambda: ops.linear_int8_grad_weight(x, dz)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)
    with pytest.raises(_native.NerfHipError):
        ops.linear_int8(rows, packed, b.cpu())


@gpu_only
def test_no_rows(gpu):
    from nerf_amd import ops
    x, w, dz, b = make(3, 70, 9, 1, gpu)
    rows, packed = ops.quantize_rows(x[:0], True, True), ops.pack_int8(w, True)
    assert rows.q.shape == (0, 128) and rows.mask.shape == (0, 16)
    assert ops.linear_int8(rows, packed, b).shape == (0, 9)
    assert ops.linear_int8_quantized(rows, packed, b).q.shape == (0, 64)
    assert ops.linear_int8_grad_input(dz[:0], packed, rows.mask).shape == (0, 70)
    dw, db = ops.linear_int8_grad_weight(rows, dz[:0])
    assert dw.shape == (70, 9) and not bool(dw.any()) and not bool(db.any())


def _layer(x, w, dz, b):
    from nerf_amd import ops
    packed, rows = ops.pack_int8(w, True), ops.quantize_rows(x, True, True)
    y = ops.linear_int8(rows, packed, b, relu=True, dtype=torch.bfloat16)
    nxt = ops.linear_int8_quantized(rows, packed, b, relu=True, pow2=True, want_mask=True)
    dw, db = ops.linear_int8_grad_weight(rows, dz)
    return [y, nxt.q, nxt.scale, nxt.mask, dw, db, ops.linear_int8_grad_input(dz, packed, rows.mask)]


@gpu_only
@pytest.mark.parametrize("n,k,m", [(700, 63, 256), (1, 256, 128), (5000, 256, 256), (4500, 320, 384), (600, 64, 800), (33000, 256, 256), (16400, 512, 512)])
def test_a_layer_on_other_streams_and_in_graphs(gpu, n, k, m):
    """Two streams at once, and two captured graphs replayed in turn on fresh inputs, with eager work between:
    the bits of the plain calls."""
    x, w, dz, b = make(n, k, m, 2, gpu)
    x2, w2, dz2, b2 = make(n, k, m, 3, gpu)
    want, want2 = _layer(x, w, dz, b), _layer(x2, w2, dz2, b2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(s1):
            got = _layer(x, w, dz, b)
        with torch.cuda.stream(s2):
            got2 = _layer(x2, w2, dz2, b2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)) and all(torch.equal(a, c) for a, c in zip(got2, want2))
    ins = [[t.clone() for t in (x, w, dz, b)] for _ in range(2)]
    graphs = []
    for i in ins:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = _layer(*i)
        graphs.append((gr, out))
    for turn in range(4):
        first, second = ((x, w, dz, b), (x2, w2, dz2, b2)) if turn % 2 else ((x2, w2, dz2, b2), (x, w, dz, b))
        for (gr, out), fresh, held in zip(graphs, (first, second), ins):
            for a, c in zip(held, fresh):
                a.copy_(c)
            gr.replay()
        eager = _layer(x, w, dz, b)
        torch.cuda.synchronize()
        for (gr, out), fresh in zip(graphs, (first, second)):
            ref = want if fresh[0] is x else want2
            assert all(torch.equal(a, c) for a, c in zip(out, ref)), turn
        assert all(torch.equal(a, c) for a, c in zip(eager, want))


@gpu_only
def test_offsets_beyond_32_bits(gpu):
    """8.5 million rows of 256 integers: 2.2 GB of rows, 4.4 GB of outputs.  The last rows are those of a small call."""
    from nerf_amd import ops
    n, k, m = 8_500_000, 256, 256
    tail = 300
    _, w, dz, b = make(tail, k, m, 4, gpu)
    x = torch.zeros((n, k), dtype=torch.bfloat16, device=gpu)
    x[-tail:] = torch.randn((tail, k), device=gpu)
    rows, packed = ops.quantize_rows(x, True, True), ops.pack_int8(w, True)
    small = ops.quantize_rows(x[-tail:], True, True)
    assert torch.equal(rows.q[-tail:], small.q) and torch.equal(rows.mask[-tail:], small.mask) and torch.equal(rows.scale[-tail:], small.scale)
    y = ops.linear_int8(rows, packed, b, relu=True, dtype=torch.bfloat16)
    assert torch.equal(y[-tail:], ops.linear_int8(small, packed, b, relu=True, dtype=torch.bfloat16))
    del y
    nxt, nxs = ops.linear_int8_quantized(rows, packed, b, True, pow2=True, want_mask=True), ops.linear_int8_quantized(small, packed, b, True, pow2=True, want_mask=True)
    assert torch.equal(nxt.q[-tail:], nxs.q) and torch.equal(nxt.scale[-tail:], nxs.scale) and torch.equal(nxt.mask[-tail:], nxs.mask)
    big = torch.zeros((n, m), dtype=torch.bfloat16, device=gpu)
    big[-tail:] = dz
    dx = ops.linear_int8_grad_input(big, packed, rows.mask)
    assert not bool(dx[:-tail].any())
    p, ws, _ = ref_linear(small, w, True)
    wd, d, xd = p * ws, big[-tail:].double(), dequantised(small)
    want, on = d @ wd.t().contiguous(), unpack_bits(small.mask, k)
    close(dx[-tail:], want * on, on * (d.abs() @ wd.abs().t().contiguous() * m * 2.0 ** -23 + 2.0 ** -8 * want.abs() + 1e-38), "dx")
    dw, db = ops.linear_int8_grad_weight(rows, big)
    close(dw, xd.t().contiguous() @ d, xd.abs().t().contiguous() @ d.abs() * tail * 2.0 ** -23 + 1e-35, "dW")
    close(db, d.sum(0), d.abs().sum(0) * tail * 2.0 ** -23 + 1e-38, "db")


@gpu_only
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,k,m", [(40, 70, 96), (5000, 100, 96), (4500, 130, 33), (4200, 64, 3), (4200, 300, 222), (4096, 256, 256), (4300, 640, 600), (4300, 640, 500), (4300, 640, 190),
                                   (32900, 300, 222), (33000, 64, 3), (32768, 256, 256), (33000, 130, 33), (16000, 640, 600)])
def test_a_row_that_is_not_finite_stays_one_row(gpu, n, k, m, dtype):
    """A NaN in one row (in the middle, in the last) reaches that row's results and no other's, whatever the
    width the rows are padded to."""
    from nerf_amd import ops
    x, w, dz, b = make(n, k, m, 9, gpu, TYPES[dtype])
    packed = ops.pack_int8(w, True)
    good = ops.linear_int8_grad_input(dz, packed)
    goody = ops.linear_int8(ops.quantize_rows(x), packed, b)
    for at in (n // 3, n - 1):
        bad, badx = dz.clone(), x.clone()
        bad[at, m // 2], badx[at, k // 2] = float("nan"), float("inf")
        dx, y = ops.linear_int8_grad_input(bad, packed), ops.linear_int8(ops.quantize_rows(badx), packed, b)
        rest = torch.arange(n, device=gpu) != at
        assert bool(torch.isnan(dx[at]).all()) and torch.equal(dx[rest], good[rest])
        assert bool(torch.isnan(y[at]).all()) and torch.equal(y[rest], goody[rest])


@gpu_only
@pytest.mark.parametrize("dt,t", [(0, torch.float32), (1, torch.float16), (2, torch.bfloat16)])
@pytest.mark.parametrize("n,k,m", [(1, 5, 3), (37, 70, 19), (4100, 283, 130), (4099, 256, 256), (4100, 65, 600), (4101, 700, 200), (4100, 65, 450), (40, 650, 300), (129, 1000, 70), (300, 1100, 1100),
                                   (32769, 283, 130), (32801, 256, 256), (33000, 65, 600), (33001, 700, 200)])
def test_nothing_else_is_written(gpu, n, k, m, dt, t):
    """The C entry points on buffers with room between and behind the rows: what is not theirs keeps its bytes."""
    from nerf_amd import _native, ops
    lib, st = _native.lib(), torch.cuda.current_stream().cuda_stream
    x, w, dz, b = make(n, k, m, 6, gpu, t)
    rows, packed = ops.quantize_rows(x, True, True), ops.pack_int8(w, True)
    kp, mp = rows.q.shape[1], -(-m // 64) * 64

    def fresh(r, c, dtype):
        return torch.full((r, c), 77, dtype=dtype, device=gpu)
    q, s, bits = fresh(n + 2, kp, torch.int8), fresh(n + 2, 1, torch.float32), fresh(n + 2, kp // 8, torch.uint8)
    assert lib.nerf_quantize_rows(x.data_ptr(), dt, n, k, k, 1, q.data_ptr(), s.data_ptr(), bits.data_ptr(), st) == 0
    assert torch.equal(q[:n], rows.q) and torch.equal(s[:n, 0], rows.scale) and torch.equal(bits[:n], rows.mask)
    assert bool((q[n:] == 77).all()) and bool((s[n:] == 77).all()) and bool((bits[n:] == 77).all())
    y = fresh(n + 2, m + 5, t)
    assert lib.nerf_linear_int8(rows.q.data_ptr(), rows.scale.data_ptr(), n, k, packed.packed.data_ptr(), m, b.data_ptr(), None, 0, 0, 1,
                                y.data_ptr(), dt, m + 5, st) == 0
    assert torch.equal(y[:n, :m], ops.linear_int8(rows, packed, b, relu=True, dtype=t))
    assert bool((y[n:] == 77).all()) and bool((y[:, m:] == 77).all())
    need = lib.nerf_linear_int8_quantized_bytes(n, m)
    ws = fresh(need + 64, 1, torch.uint8)
    yq, ys, yb = fresh(n + 2, mp, torch.int8), fresh(n + 2, 1, torch.float32), fresh(n + 2, mp // 8, torch.uint8)
    assert lib.nerf_linear_int8_quantized(rows.q.data_ptr(), rows.scale.data_ptr(), n, k, packed.packed.data_ptr(), m, b.data_ptr(), None, 0,
                                          0, 1, 1, yq.data_ptr(), ys.data_ptr(), yb.data_ptr(), ws.data_ptr(), need, st) == 0
    ref = ops.linear_int8_quantized(rows, packed, b, relu=True, pow2=True, want_mask=True)
    assert torch.equal(yq[:n], ref.q) and torch.equal(ys[:n, 0], ref.scale) and torch.equal(yb[:n], ref.mask)
    assert bool((yq[n:] == 77).all()) and bool((ys[n:] == 77).all()) and bool((yb[n:] == 77).all()) and bool((ws[need:] == 77).all())
    dx = fresh(n + 2, k + 3, t)
    assert lib.nerf_linear_int8_grad_input(dz.data_ptr(), dt, n, m, m, packed.packed.data_ptr(), k, rows.mask.data_ptr(), dx.data_ptr(), k + 3, st) == 0
    assert torch.equal(dx[:n, :k], ops.linear_int8_grad_input(dz, packed, rows.mask))
    assert bool((dx[n:] == 77).all()) and bool((dx[:, k:] == 77).all())
    need = lib.nerf_linear_int8_grad_weight_bytes(n, k, m)
    dw, db, ws = fresh(k + 1, m, torch.float32), fresh(m + 3, 1, torch.float32), fresh(need + 64, 1, torch.uint8)
    assert lib.nerf_linear_int8_grad_weight(rows.q.data_ptr(), rows.scale.data_ptr(), n, k, dz.data_ptr(), dt, m, m, dw.data_ptr(), db.data_ptr(),
                                            ws.data_ptr(), need, st) == 0
    ref = ops.linear_int8_grad_weight(rows, dz)
    assert torch.equal(dw[:k], ref[0]) and torch.equal(db[:m, 0], ref[1])
    assert bool((dw[k:] == 77).all()) and bool((db[m:] == 77).all()) and bool((ws[need:] == 77).all())
    packed2 = fresh(packed.packed.numel() + 64, 1, torch.uint8)
    assert lib.nerf_int8_pack(w.data_ptr(), k, m, 1, packed2.data_ptr(), st) == 0
    assert torch.equal(packed2[:-64, 0], packed.packed) and bool((packed2[-64:] == 77).all())
