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
