"""Networks of other depths and widths on the 8-bit layers: init_nerf_model(precision='int8')."""
import numpy as np
import pytest
import torch

from tests.test_int8_layers import TYPES, close, dequantised, ref_linear, unpack_bits  # noqa: F401
from tests.util import default_args, pose_spherical

gpu_only = pytest.mark.gpu
SHAPE = dict(D=3, W=40, input_ch=21, input_ch_views=9, output_ch=4, skips=[1], use_viewdirs=True)


def test_shapes_are_checked_without_a_gpu():
    from nerf_amd.layered import LayeredNerfModel
    from nerf_amd.run_nerf_helpers import NerfModel, init_nerf_model
    m = init_nerf_model(**SHAPE, device="cpu", precision='int8')
    assert isinstance(m, LayeredNerfModel) and m.layered and not NerfModel.layered
    assert m.shapes == [(21, 40), (40, 40), (61, 40), (40, 256), (265, 20), (20, 3), (40, 1)]
    assert [m.split(i) for i in range(7)] == [[(0, 21, True)], [(0, 40, False)], [(0, 21, True), (21, 40, False)], [(0, 40, False)],
                                              [(0, 256, False), (256, 9, True)], [(0, 20, False)], [(0, 40, False)]]
    ws = [w.copy() for w in m.get_weights()]
    m.set_weights([w + 1 for w in ws])
    assert all(np.array_equal(a, b + 1) for a, b in zip(m.get_weights(), ws))
    with pytest.raises(NotImplementedError):
        m.packed()
    for bad in (dict(D=0), dict(W=1), dict(W=5000), dict(input_ch=20), dict(use_viewdirs=False), dict(output_ch=5), dict(skips=[-1])):
        with pytest.raises(NotImplementedError):
            init_nerf_model(**{**SHAPE, **bad}, device="cpu", precision='int8')
    with pytest.raises(ValueError):
        init_nerf_model(**SHAPE, device="cpu", precision='int4')
    with pytest.raises(NotImplementedError):
        init_nerf_model(**SHAPE, device="cpu")


def _net(gpu, seed=0, **change):
    from nerf_amd.run_nerf_helpers import init_nerf_model
    g = torch.Generator(device=gpu).manual_seed(seed)
    m = init_nerf_model(**{**SHAPE, **change}, device=gpu, generator=g, precision='int8')
    with torch.no_grad():
        for i in range(len(m.shapes)):
            m.bias(i).copy_(0.1 * torch.randn(m.bias(i).shape, generator=g, device=gpu))
    m.mark_dirty()
    return m


@gpu_only
@pytest.mark.parametrize("change", [dict(), dict(D=8, W=256, input_ch=63, input_ch_views=27, skips=[4]), dict(D=2, W=130, skips=[1]),
                                    dict(D=1, W=7, input_ch=3, input_ch_views=3, skips=[]), dict(D=4, W=300, skips=[0, 2])])
def test_forward_and_gradients_layer_by_layer(gpu, change):
    """Every layer's integers from the layer's own recorded input, and every gradient from the recorded
    integers and masks, in 64 bits.  The bound of a gradient follows the rounding of dz to bf16 (2^-9) and
    the fp32 sums (c 2^-23) through the layers."""
    from nerf_amd import ops
    from nerf_amd.layered import _Pass
    net = _net(gpu, **change)
    n, S = 23, 7
    g = torch.Generator(device=gpu).manual_seed(1)
    pts = torch.rand((n * S, 3), generator=g, device=gpu) * 2 - 1
    vd = torch.nn.functional.normalize(torch.randn((n, 3), generator=g, device=gpu), dim=1)
    run = _Pass(net, pts, vd, S)
    D = net.D
    W = [[ref_linear(rows, net.weight(i)[r0:r0 + k].detach(), True)[:2] for rows, (r0, k, _) in zip(run.inputs[i], net.split(i))]
         for i in range(len(net.shapes))]
    W = [[p * s for p, s in parts] for parts in W]                                   # as the products used them
    pe = net.input_ch if net.input_ch == 3 else ops.embed(pts, (net.input_ch - 3) // 6)
    first = ops.quantize_rows(pts if net.input_ch == 3 else pe, pow2=True)
    assert torch.equal(run.inputs[0][0].q, first.q) and torch.equal(run.inputs[0][0].scale, first.scale)

    def before_relu(i):
        parts = [dequantised(r) @ w for r, w in zip(run.inputs[i], W[i])]
        mag = sum(dequantised(r).abs() @ w.abs() for r, w in zip(run.inputs[i], W[i]))
        z = sum(parts) + net.bias(i).detach().double()
        # the encoding's part goes through bf16 (half a step: 2^-9), everything through a few fp32 roundings
        tol = sum(p.abs() * 2.0 ** -8 for p, (_, _, enc) in zip(parts, net.split(i)) if enc and len(parts) > 1) + (mag + z.abs()) * 2.0 ** -21
        return z, tol
    for i, out in [(i, run.inputs[i + 1][-1]) for i in range(D - 1)] + [(D - 1, run.inputs[D][-1]), (D, run.inputs[D + 1][0]), (D + 1, run.inputs[D + 2][0])]:
        z, tol = before_relu(i)
        y = z if i == D else z.clamp(min=0)
        if i != D:
            on = unpack_bits(out.mask, out.k)
            assert not bool((on != (z > 0))[z.abs() > tol].any())
        # half a step of the row's scale, which is the next power of two of its largest value
        close(dequantised(out), y, tol + 0.5 * out.scale.double()[:, None] * (1 + 1e-6), (i, change))
        top = y.abs().amax(1)
        assert bool((out.scale.double() * 127 * (1 + 1e-5) + tol.max() >= top).all())
        assert bool((out.scale.double() * 127 / 2 <= top * (1 + 1e-5) + tol.max() + 1e-30).all())
    rgb, tol = before_relu(D + 2)
    close(run.raw[:, :3], rgb, tol + 1e-30, "rgb")
    alpha, tol = before_relu(D + 3)
    close(run.raw[:, 3:], alpha, tol + 1e-30, "alpha")

    d_raw = torch.randn((n * S, 4), generator=g, device=gpu) * 10.0 ** (-3 * torch.rand((n * S, 1), generator=g, device=gpu))
    got = run.gradients(d_raw)
    d = d_raw.double()
    ok = lambda x, y, b, what: close(x, y, b * 1.001 + 1e-35, (what, change))

    def check(i, dz, err):
        x = torch.cat([dequantised(r) for r in run.inputs[i]], 1)
        c = 3 * n * S * 2.0 ** -23
        ok(got[2 * i], x.t().contiguous() @ dz, x.abs().t().contiguous() @ (err + c * (dz.abs() + err)), f"W {i}")
        ok(got[2 * i + 1], dz.sum(0), (err + c * (dz.abs() + err)).sum(0), f"b {i}")

    def back(i, dz, err, mask=True):
        at = [j for j, (_, _, enc) in enumerate(net.split(i)) if not enc][0]
        w = W[i][at].t().contiguous()
        out, mag = dz @ w, (dz.abs() + err) @ w.abs()
        e = err @ w.abs() + 2.0 ** -22 * dz.shape[1] * mag
        e = e + 2.0 ** -9 * (out.abs() + e)
        if mask:
            on = unpack_bits(run.inputs[i][at].mask, w.shape[1])
            out, e = out * on, e * on
        return out, e
    exact = torch.zeros_like(d)
    half = 2.0 ** -9 * d.abs()                                     # d raw itself goes back in bf16
    check(D + 2, d[:, :3], exact[:, :3])
    check(D + 3, d[:, 3:], exact[:, 3:])
    dz, err = back(D + 2, d[:, :3], half[:, :3])
    check(D + 1, dz, err)
    dz, err = back(D + 1, dz, err, mask=False)
    check(D, dz, err)
    a, ea = back(D, dz, err)
    b, eb = back(D + 3, d[:, 3:], half[:, 3:])
    dz, err = a + b, ea + eb
    err = err + 2.0 ** -9 * (dz.abs() + err)
    for i in range(D - 1, -1, -1):
        check(i, dz, err)
        if i:
            dz, err = back(i, dz, err)


def _args(**change):
    a = default_args()
    for k, v in dict(precision='int8', netdepth=3, netwidth=48, netdepth_fine=4, netwidth_fine=64, multires=4, multires_views=2,
                     N_samples=12, N_importance=9, no_reload=True, perturb=1.0, **change).items():
        setattr(a, k, v)
    return a


@gpu_only
def test_create_nerf_render_and_query(gpu, tmp_path):
    from nerf_amd import checkpoint, ops
    from nerf_amd.run_nerf import create_nerf, render
    a = _args()
    torch.manual_seed(0)
    kw_train, kw_test, start, grad_vars, models = create_nerf(a)
    assert models['model'].layered and models['model_fine'].D == 4 and len(grad_vars) == 2 * (3 + 4) + 2 * (4 + 4)
    H = W = 10
    c2w = torch.as_tensor(pose_spherical(30., -30., 4.)[:3, :4].astype(np.float32))
    out = render(H, W, 9.0, chunk=64, c2w=c2w, near=2., far=6., retraw=True, **kw_test)
    rgb, disp, acc, extras = out
    assert rgb.shape == (H, W, 3) and extras['raw'].shape == (H, W, 21, 4) and bool(torch.isfinite(rgb).all())
    again = render(H, W, 9.0, chunk=100000, c2w=c2w, near=2., far=6., retraw=True, **kw_test)
    assert torch.equal(again[0], rgb) and torch.equal(again[3]['raw'], extras['raw'])       # whatever the chunk
    # the query closure on explicit points: the points and directions of one ray are the render's
    o, d = ops.get_rays(H, W, 9.0, c2w)
    rays = ops.build_ray_batch(o, d, d, False, H, W, 9.0, 2., 6.)
    z = ops.sample_z(rays, 12)
    pts = rays[:, None, 0:3] + rays[:, None, 3:6] * z[:, :, None]
    raw = kw_test['network_query_fn'](pts, rays[:, 8:11], models['model'])
    assert raw.shape == (H * W, 12, 4)
    flat = kw_test['network_query_fn'](pts[:, 0], rays[:, 8:11], models['model'])
    assert torch.equal(flat, raw[:, 0])
    with pytest.raises(ValueError):
        kw_test['network_query_fn'](pts, rays[:5, 8:11], models['model'])
    # a checkpoint holds the same arrays in the same order
    path = checkpoint.save_weights(models['model'], 'model', 7, str(tmp_path), 'exp')
    net = _net(gpu, D=3, W=48, input_ch=27, input_ch_views=15, skips=[])
    net = type(net)(3, 48, 27, 15, 4, models['model'].skips, True, device=gpu)
    net.set_weights(checkpoint.load_weights(path))
    assert torch.equal(kw_test['network_query_fn'](pts, rays[:, 8:11], net), raw)


@gpu_only
def test_train_steps_plain_and_graphed(gpu):
    """train_step and GraphedTrainStep: the same bits, weights that move, a loss that is finite; and the
    recorded forward pass gives the bits of the one that is not."""
    from nerf_amd import training
    from nerf_amd.run_nerf import create_nerf, render
    runs = []
    for graphed in (False, True):
        torch.manual_seed(3)
        a = _args()
        kw_train, kw_test, start, grad_vars, models = create_nerf(a)
        kw_train['perturb'] = 0.                     # a captured graph draws other uniforms than eager calls
        nets = [models['model'], models['model_fine']]
        opt = training.Adam(training.ExponentialDecay(5e-4, 1000, 0.1)).bind_models(nets)
        fn = lambda r: render(8, 8, 9.0, chunk=1024, rays=r, near=2., far=6., retraw=True, **kw_train)
        g = torch.Generator(device=gpu).manual_seed(5)
        steps = training.GraphedTrainStep(fn, 33, grad_vars, opt, nets) if graphed else None
        start_w = [n.flat.clone() for n in nets]
        log = []
        for i in range(4):
            o = torch.nn.functional.normalize(torch.randn((33, 3), generator=g, device=gpu), dim=1) * 4
            d = -o / 4 + 0.1 * torch.randn((33, 3), generator=g, device=gpu)
            t = torch.rand((33, 3), generator=g, device=gpu)
            loss, _, _ = steps((o, d), t) if graphed else training.train_step(fn, (o, d), t, grad_vars, opt)
            log.append(loss.detach().clone())
            fresh = fn((o, d))[0]                    # eager work between the steps, with the new weights
            assert bool(torch.isfinite(fresh).all())
        assert all(bool(torch.isfinite(l)) for l in log) and all(not torch.equal(n.flat, w) for n, w in zip(nets, start_w))
        runs.append((torch.stack(log), [n.flat.detach().clone() for n in nets]))
    assert torch.equal(runs[0][0], runs[1][0]) and all(torch.equal(x, y) for x, y in zip(runs[0][1], runs[1][1]))
    with training.GradientTape():
        rec = fn((o, d))
    plain = fn((o, d))
    assert torch.equal(rec[0].detach(), plain[0]) and torch.equal(rec[3]['raw'].detach(), plain[3]['raw'])


@gpu_only
@pytest.mark.parametrize("precision", ['int8', None])
def test_a_step_captured_while_an_eager_graph_lives(gpu, precision):
    """The outputs of an eager tape over the same parameters, still held, do not disturb a capture: its leaves are its own."""
    from nerf_amd import training
    from nerf_amd.run_nerf import create_nerf, render
    runs = []
    for graphed in (False, True):
        torch.manual_seed(4)
        a = _args() if precision else default_args()
        a.precision, a.N_samples, a.N_importance, a.no_reload = precision, 12, 9, True
        kw_train, _, _, grad_vars, models = create_nerf(a)
        kw_train['perturb'] = 0.
        nets = [models['model'], models['model_fine']]
        opt = training.Adam(5e-4).bind_models(nets)
        fn = lambda r: render(8, 8, 9.0, chunk=1024, rays=r, near=2., far=6., retraw=True, **kw_train)
        g = torch.Generator(device=gpu).manual_seed(6)
        o = torch.nn.functional.normalize(torch.randn((32, 3), generator=g, device=gpu), dim=1) * 4
        t = torch.rand((32, 3), generator=g, device=gpu)
        with training.GradientTape():
            held = fn((o, -o / 4))                   # ... and its graph with it
        params = [list(n.params) for n in nets]
        step = training.GraphedTrainStep(fn, 32, grad_vars, opt, nets) if graphed else None
        for _ in range(3):
            step((o, -o / 4), t) if graphed else training.train_step(fn, (o, -o / 4), t, grad_vars, opt)
        assert all(p is q for n, ps in zip(nets, params) for p, q in zip(n.params, ps)) and held[0].grad_fn is not None
        runs.append([n.flat.detach().clone() for n in nets])
    assert all(torch.equal(x, y) for x, y in zip(*runs))


@gpu_only
def test_two_queries_of_one_network_and_unused_ones(gpu):
    """The coarse network doing the fine pass too: autograd adds both contributions; an output that does not
    reach the loss costs nothing."""
    from nerf_amd import training
    from nerf_amd.layered import LayeredQuery
    net = _net(gpu)
    g = torch.Generator(device=gpu).manual_seed(2)
    rays = torch.rand((9, 11), generator=g, device=gpu)
    z = [torch.rand((9, s), generator=g, device=gpu).sort(1).values for s in (4, 6)]
    w = [torch.randn((9, s, 4), generator=g, device=gpu) for s in (4, 6)]
    with training.GradientTape() as tape:
        a, b = (LayeredQuery.apply(rays, x, net, *net.params) for x in z)
        both = tape.gradient((a * w[0]).sum() + (b * w[1]).sum(), net.params)
    parts = []
    for x, y in zip(z, w):
        with training.GradientTape() as tape:
            q = LayeredQuery.apply(rays, x, net, *net.params)
            LayeredQuery.apply(rays, x, net, *net.params)
            parts.append(tape.gradient((q * y).sum(), net.params))
    assert all(torch.equal(t, p + q) for t, p, q in zip(both, *parts))


@gpu_only
def test_backward_passes_that_cannot_be_right_raise(gpu):
    from nerf_amd import training
    from nerf_amd.layered import LayeredQuery
    net = _net(gpu)
    rays = torch.rand((9, 11), device=gpu)
    z = torch.rand((9, 4), device=gpu).sort(1).values
    with training.GradientTape():
        raw = LayeredQuery.apply(rays, z, net, *net.params)
        torch.autograd.grad(raw.sum(), net.params, retain_graph=True)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(raw.sum(), net.params)
        raw = LayeredQuery.apply(rays, z, net, *net.params)
        net.set_weights([w * 2 for w in net.get_weights()])
        with pytest.raises(RuntimeError, match="changed"):
            torch.autograd.grad(raw.sum(), net.params)
        raw = LayeredQuery.apply(rays, z, net, *net.params)       # ... and the network is as good as before
        assert all(bool(torch.isfinite(g).all()) for g in torch.autograd.grad(raw.sum(), net.params))


@gpu_only
@pytest.mark.parametrize("n,S", [(0, 5), (3, 0), (0, 0)])
def test_no_points(gpu, n, S):
    from nerf_amd.run_nerf import create_nerf
    kw = create_nerf(_args())[1]
    raw = kw['network_query_fn'](torch.zeros((n, S, 3), device=gpu), torch.zeros((n, 3), device=gpu), kw['network_fn'])
    assert raw.shape == (n, S, 4)


def _alone_over_rccl(rank, port, tmp):
    import os
    import torch.distributed as dist
    from nerf_amd import parallel, training
    from nerf_amd.run_nerf import create_nerf, render
    torch.cuda.set_device(0)
    gpu = torch.device("cuda", 0)
    try:
        dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1, device_id=gpu)
        dist.all_reduce(torch.ones(4, device=gpu))
        torch.cuda.synchronize()
    except Exception as e:  # no RCCL on this machine: nothing to test
        open(os.path.join(tmp, "unavailable"), "w").write(repr(e))
        return
    try:
        def run(exchange):
            parallel.EXCHANGE_WHEN_ALONE = exchange
            torch.manual_seed(9)
            kw_train, _, _, grad_vars, models = create_nerf(_args())
            nets = [models['model'], models['model_fine']]
            opt = training.Adam(5e-4).bind_models(nets)
            g = torch.Generator(device=gpu).manual_seed(5)
            o = torch.nn.functional.normalize(torch.randn((64, 3), generator=g, device=gpu), dim=1) * 4
            t = torch.rand((64, 3), generator=g, device=gpu)
            fn = lambda r: render(8, 8, 9.0, chunk=1024, rays=r, near=2., far=6., retraw=True, **{**kw_train, 'perturb': 0.})
            losses = [training.train_step(fn, (o, -o / 4), t, grad_vars, opt)[0] for _ in range(3)]
            return torch.stack(losses), [n.flat.detach().clone() for n in nets]
        plain, over = run(False), run(True)
        assert torch.equal(plain[0], over[0]) and all(torch.equal(a, b) for a, b in zip(plain[1], over[1]))
        open(os.path.join(tmp, "ok"), "w").write("ok")
    finally:
        parallel.EXCHANGE_WHEN_ALONE = False
        dist.destroy_process_group()


@gpu_only
def test_data_parallel_step_over_rccl_with_one_rank(gpu, tmp_path):
    """The exchanges of one rank are identities (64 rays: the ray-count weight is a power of two)."""
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    torch.multiprocessing.spawn(_alone_over_rccl, args=(port, str(tmp_path)), nprocs=1, join=True)
    if (tmp_path / "unavailable").exists():
        pytest.skip((tmp_path / "unavailable").read_text())
    assert (tmp_path / "ok").exists()
