"""Layered networks outside training: what they refuse, the memory a query takes, the order of streams, accuracy."""
import pytest
import torch

SHAPE = dict(D=3, W=40, input_ch=21, input_ch_views=9, output_ch=4, skips=[1], use_viewdirs=True)


def test_the_fused_streams_of_a_layered_network_are_refused():
    """Its layers are other shapes than the fused layouts read, also where there are as many."""
    from nerf_amd.run_nerf_helpers import init_nerf_model
    for D in (3, 8):
        net = init_nerf_model(**{**SHAPE, 'D': D}, device="cpu", precision='int8')
        for call in (net.packed, net.packed_bwd):
            with pytest.raises(NotImplementedError, match="layered"):
                call()


# ---- memory of a query ----------------------------------------------------------------------------------
@pytest.mark.parametrize("P,S,most", [(0, 5, 7), (12, 4, 100), (12, 4, 12), (12, 4, 11), (12, 4, 4), (12, 4, 3), (12, 4, 1), (1000, 1, 64), (777, 777, 100), (2100, 700, 333)])
def test_pieces_of_a_query(P, S, most):
    """Every point once and in order, with its ray, and no piece larger than asked for."""
    from nerf_amd.layered import _pieces
    at = 0
    for a, b, ray, s in _pieces(P, S, most):
        assert a == at and 0 < b - a <= most and (b - a) % s == 0
        assert all((p - a) // s + ray == p // S for p in range(a, b))
        at = b
    assert at == P


@pytest.mark.parametrize("change,points", [(dict(D=8, W=256, input_ch=63, input_ch_views=27, skips=[4]), 1 << 20), (dict(D=2, W=2, skips=[]), 1 << 20),
                                           (dict(D=64, W=4096, skips=[]), None), (dict(D=1, W=4096, input_ch=63, skips=[0]), None)])
def test_the_points_of_a_query_go_by_the_widest_layer(change, points, monkeypatch):
    from nerf_amd import layered
    # (without the parameters, which a 64 x 4096 network has 4 GiB of)
    net = type('Net', (), dict(split=layered.LayeredNerfModel.split))()
    s = {**SHAPE, **change}
    net.D, net.W, net.input_ch, net.input_ch_views, net.skips = s['D'], s['W'], s['input_ch'], s['input_ch_views'], s['skips']
    k, net.shapes = net.input_ch, []
    for i in range(net.D):
        net.shapes.append((k, net.W))
        k = net.W + (net.input_ch if i in net.skips else 0)
    net.shapes += [(k, 256), (256 + net.input_ch_views, net.W // 2), (net.W // 2, 3), (k, 1)]
    got = layered.query_points(net)
    assert points is None or got == points
    # two rows of integers and an fp32 row of the widest layer are below the bound, and the budget above it
    assert layered.point_bytes(net) >= 2 * net.W + 4 * net.W and got * layered.point_bytes(net) <= layered._QUERY_BYTES
    monkeypatch.setattr(layered, '_QUERY_BYTES', 1)
    assert layered.query_points(net) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("change", [dict(D=12, W=700, skips=[3]), dict(D=5, W=256, input_ch=63, input_ch_views=27, skips=[0, 2]), dict(D=3, W=1100, skips=[])])
def test_a_query_stays_within_its_memory(gpu, change, monkeypatch):
    """The peak of a query, beside its result and a piece of fragments, is within the bytes that it is given, whatever the
    depth; its result is that of one piece, and of a pass that records."""
    from nerf_amd import layered
    from nerf_amd.run_nerf_helpers import init_nerf_model
    net = init_nerf_model(**{**SHAPE, **change}, device=gpu, generator=torch.Generator(device=gpu).manual_seed(7), precision='int8')
    n, S = 4000, 9
    pts = torch.rand((n * S, 3), device=gpu) * 2 - 1
    vd = torch.nn.functional.normalize(torch.randn((n, 3), device=gpu), dim=1)
    want = layered._Pass(net, pts, vd, S).raw
    assert torch.equal(layered.query(net, pts, vd, S), want)
    budget = 16 << 20
    monkeypatch.setattr(layered, '_QUERY_BYTES', budget)
    assert layered.query_points(net) < n * S / 3
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = layered.query(net, pts, vd, S)
    peak = torch.cuda.max_memory_allocated() - before - got.numel() * 4
    assert torch.equal(got, want)
    assert peak <= budget + (1 << 20), (peak, layered.query_points(net), layered.point_bytes(net))   # (blocks are rounded to 512 bytes)
    monkeypatch.setattr(layered, '_QUERY_BYTES', 4 * layered.point_bytes(net))                       # parts of one ray
    assert torch.equal(layered.query(net, pts[:5 * S], vd[:5], S), want[:5 * S])


# ---- streams ---------------------------------------------------------------------------------------
def _rays(gpu, n, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.rand((n, 11), generator=g, device=gpu), torch.rand((n, 6), generator=g, device=gpu).sort(1).values


def _networks(gpu, precision):
    """A network and one with other weights of the same shape; and its forward pass."""
    from nerf_amd import layered, ops
    from nerf_amd.run_nerf_helpers import init_nerf_model
    shape = SHAPE if precision else dict(D=8, W=256, input_ch=63, input_ch_views=27, output_ch=4, skips=[4], use_viewdirs=True)
    nets = [init_nerf_model(**shape, device=gpu, generator=torch.Generator(device=gpu).manual_seed(s), precision=precision) for s in (0, 1)]

    def query(net, rays, z):
        if not precision:
            return ops.mlp_forward_rays(net.packed(), rays, z)
        pts = (rays[:, None, 0:3] + rays[:, None, 3:6] * z[:, :, None]).reshape(-1, 3)
        return layered.query(net, pts, rays[:, 8:11].contiguous(), z.shape[1]).view(*z.shape, 4)
    return nets, query


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ['int8', None])
def test_two_streams_query_one_network_that_has_just_changed(gpu, precision):
    """The parameters have changed for both streams; the first one to query lays them out, behind other work of its own;
    the second must not read the memory before that."""
    (net, other), query = _networks(gpu, precision)
    rays, z = _rays(gpu, 50, 3)
    want = query(other, rays, z)
    query(net, rays, z)                                     # what the memory holds before
    net.set_weights(other.get_weights())
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        torch.cuda._sleep(20_000_000)                       # some ten milliseconds
        a = query(net, rays, z)
    with torch.cuda.stream(second):
        b = query(net, rays, z)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)
    c = query(net, rays, z)
    torch.cuda.synchronize()
    assert torch.equal(c, want)


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ['int8', None])
def test_two_host_threads_query_one_network_that_has_just_changed(gpu, precision):
    import threading
    (net, other), query = _networks(gpu, precision)
    rays, z = _rays(gpu, 40, 6)
    want = [query(m, rays, z) for m in (net, other)]
    weights = [[w.copy() for w in m.get_weights()] for m in (net, other)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(8):
        net.set_weights(weights[(turn + 1) % 2])
        torch.cuda.synchronize()
        start, got = threading.Barrier(2), [None, None]

        def work(i):
            torch.cuda.set_device(gpu)
            with torch.cuda.stream(streams[i]):
                start.wait()
                got[i] = query(net, rays, z)
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert all(torch.equal(a, want[(turn + 1) % 2]) for a in got)


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ['int8', None])
def test_a_copied_network_lays_out_its_own_weights(gpu, precision):
    import copy
    (net, other), query = _networks(gpu, precision)
    rays, z = _rays(gpu, 20, 4)
    want, held = query(other, rays, z), query(net, rays, z)
    twin = copy.deepcopy(net)
    twin.set_weights(other.get_weights())
    assert torch.equal(query(twin, rays, z), want) and torch.equal(query(net, rays, z), held)


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ['int8', None])
def test_weights_laid_out_in_a_capture_are_not_there_yet(gpu, precision):
    """A query captured when the parameters have just changed lays them out at every replay; until the first one, calls
    outside of the graph do it themselves.  Every replay follows the parameters."""
    (net, other), query = _networks(gpu, precision)
    rays, z = _rays(gpu, 30, 5)
    old, want = query(net, rays, z), query(other, rays, z)
    weights = [[w.copy() for w in m.get_weights()] for m in (net, other)]
    net.set_weights(weights[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = query(net, rays, z)
    assert torch.equal(query(net, rays, z), want)           # eager, before any replay
    for turn in range(4):
        net.set_weights(weights[turn % 2])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want if turn % 2 else old)
        assert torch.equal(query(net, rays, z), want if turn % 2 else old)


# ---- accuracy -------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("W", [40, 256, 600])
def test_a_concatenated_layer_adds_its_parts_in_32_bits(gpu, W):
    """The density head behind a skip has the encoding and a layer as inputs and leaves fp32: against 64 bits, from the
    integers it read.  Each part: the sum and two scales, three roundings of 2^-24 of it; bias and addend one more each."""
    from nerf_amd.layered import _Pass
    from nerf_amd.run_nerf_helpers import init_nerf_model
    from tests.test_int8_layers import close, dequantised, ref_linear
    net = init_nerf_model(**{**SHAPE, 'D': 2, 'W': W, 'skips': [1]}, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1), precision='int8')
    pts = torch.rand((500, 3), device=gpu) * 2 - 1
    run = _Pass(net, pts, torch.nn.functional.normalize(torch.randn((100, 3), device=gpu), dim=1), 5)
    head = net.D + 3
    assert [enc for _, _, enc in net.split(head)] == [True, False]
    want = net.bias(head).detach().double()
    mag = want.abs()
    for rows, (r0, k, _) in zip(run.inputs[head], net.split(head)):
        p, s, _ = ref_linear(rows, net.weight(head)[r0:r0 + k].detach(), True)
        want = want + dequantised(rows) @ (p * s)
        mag = mag + (dequantised(rows) @ (p * s)).abs()
    close(run.raw[:, 3:], want, 5.001 * 2.0 ** -24 * mag, "alpha")


def _float_network(net, pe, ve):
    """(raw, variance) of the network on 64-bit parameters and encodings, and the variance of raw that its 8-bit layers'
    roundings give if they are independent: a step s has s^2 / 12, for the rows (the next power of two of their largest
    value over 127) and for the channels of W."""
    def step2(x, dim):
        top = x.abs().amax(dim, keepdim=True)
        return torch.exp2(torch.ceil(torch.log2((top / 127).clamp_min(2.0 ** -126)))) ** 2 / 12

    def layer(i, parts):
        z, var = net.bias(i).detach().double().to(pe.device), 0
        for (x, vx), (r0, k, _) in zip(parts, net.split(i)):
            w = net.weight(i)[r0:r0 + k].detach().double().to(pe.device)
            vw = step2(w, 0).expand_as(w)
            z = z + x @ w
            var = var + vx @ (w * w + vw) + (x * x) @ vw
        return z, var

    def rows(z, var):
        return z, var + step2(z, 1)

    def relu(z, var):
        return z.clamp(min=0), var * (z > 0)
    e, v = rows(pe, torch.zeros_like(pe)), rows(ve, torch.zeros_like(ve))
    h = [e]
    for i in range(net.D):
        y = rows(*relu(*layer(i, h)))
        h = [e, y] if i in net.skips else [y]
    a, va = layer(net.D + 3, h)
    y = rows(*relu(*layer(net.D + 1, [rows(*layer(net.D, h)), v])))
    c, vc = layer(net.D + 2, [y])
    return torch.cat([c, a], 1), torch.cat([vc, va], 1)


def _points(n, far, seed, device):
    g = torch.Generator().manual_seed(seed)
    pts = (torch.rand((n, 3), generator=g) * 2 - 1) * far
    vd = torch.nn.functional.normalize(torch.randn((n, 3), generator=g), dim=1)
    return pts.to(device), vd.to(device)


def _encoded(x, channels):
    x = x.double()
    return torch.cat([x] + [f(x * 2.0 ** i) for i in range((channels - 3) // 6) for f in (torch.sin, torch.cos)], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [0.5, 2.0, 6.0])
@pytest.mark.parametrize("change", [dict(D=8, W=256, input_ch=63, input_ch_views=27, skips=[4]), dict(D=4, W=128, skips=[0, 3]), dict(D=3, W=640)])
def test_the_network_as_a_whole_is_off_by_its_roundings(gpu, change, far):
    """Against the same network in 64 bits: what 8-bit rows and weights of the stated steps give, taken as independent;
    twice that, for what they have in common (a row's or a channel's errors share a scale, points share the weights)."""
    from nerf_amd import layered
    from nerf_amd.run_nerf_helpers import init_nerf_model
    net = init_nerf_model(**{**SHAPE, **change}, device=gpu, generator=torch.Generator(device=gpu).manual_seed(11), precision='int8')
    pts, vd = _points(3000, far, 12, gpu)
    want, var = _float_network(net, _encoded(pts, net.input_ch), _encoded(vd, net.input_ch_views))
    err = layered.query(net, pts, vd, 1).double() - want
    rms, expected = err.pow(2).mean(0).sqrt(), var.mean(0).sqrt()
    assert bool((rms <= 2 * expected).all()), (rms / expected).tolist()
