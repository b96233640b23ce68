"""GraphedTrainStep: what a capture does with the networks it is given."""
import pytest
import torch

SHAPE = dict(D=2, W=8, input_ch=3, input_ch_views=3, output_ch=4, skips=[], use_viewdirs=True)


def _step(capture, models, grad_vars=None):
    """A GraphedTrainStep over networks in host memory whose capture is `capture(step)`."""
    from nerf_amd import training

    class Step(training.GraphedTrainStep):
        def _capture_on_leaves(self):
            capture(self)
    return Step(None, 4, grad_vars if grad_vars is not None else [p for m in models for p in m.params], None, models)


def _net():
    from nerf_amd.run_nerf_helpers import init_nerf_model
    return init_nerf_model(**SHAPE, device="cpu", precision='int8')


@pytest.mark.parametrize("twice", [False, True])
def test_a_capture_runs_on_leaves_and_leaves_the_parameters_in_place(twice):
    """... also where one network is listed for both passes, and where the capture fails."""
    net, other = _net(), _net()
    models = [net, net] if twice else [net, other]
    params = [list(m.params) for m in models]
    seen = []

    def capture(step):
        for m, ps in zip(models, params):
            assert all(a is not b and a.data_ptr() == b.data_ptr() and a.is_leaf and a.requires_grad for a, b in zip(m.params, ps))
        assert [l.data_ptr() for l in step._leaves] == [v.data_ptr() for v in step.grad_vars]
        assert {id(l) for l in step._leaves} == {id(p) for m in models for p in m.params}
        seen.append(len(step.models))
        if len(seen) == 2:
            raise RuntimeError("no capture")
    step = _step(capture, models)
    step._capture()
    with pytest.raises(RuntimeError, match="no capture"):
        step._capture()
    assert seen == [1 if twice else 2] * 2
    assert all(a is b for m, ps in zip(models, params) for a, b in zip(m.params, ps))


def test_hooks_of_parameters_take_part_in_a_capture():
    """A hook on a parameter changes the gradient that tape.gradient returns; it does so on the capture's leaves too,
    in the order of registration, and a removed one does not."""
    net = _net()
    calls, out = [], []
    net.params[0].register_hook(lambda g: g * 3)
    net.params[0].register_hook(lambda g: g + 1)
    net.params[2].register_hook(lambda g: calls.append(float(g.sum())))
    net.params[4].register_hook(lambda g: g * 0).remove()

    def capture(step):
        from nerf_amd import training
        with training.GradientTape() as tape:
            loss = sum((p * (i + 1)).sum() for i, p in enumerate(net.params))
        out.append(tape.gradient(loss, step._leaves))
    _step(capture, [net])._capture()
    want = [torch.full_like(p, i + 1.) for i, p in enumerate(net.params)]
    want[0] = want[0] * 3 + 1
    assert all(torch.equal(a, b) for a, b in zip(out[0], want)) and calls == [3. * net.params[2].numel()]


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ['int8', None])
def test_one_network_for_both_passes_captured(gpu, precision):
    """... listed once and twice, with a hook that halves a gradient: the bits of train_step."""
    from nerf_amd import training
    from nerf_amd.run_nerf import create_nerf, render
    from tests.util import default_args
    runs = []
    for listed in (0, 1, 2):
        torch.manual_seed(8)
        a = default_args()
        a.precision, a.N_samples, a.N_importance, a.no_reload = precision, 12, 9, True
        kw = {**create_nerf(a)[0], 'perturb': 0., 'network_fine': None}
        net = kw['network_fn']
        opt = training.Adam(5e-4).bind_models([net])
        net.params[2].register_hook(lambda g: g * 0.5)
        fn = lambda r: render(8, 8, 9.0, chunk=1024, rays=r, near=2., far=6., retraw=True, **kw)
        g = torch.Generator(device=gpu).manual_seed(9)
        step = training.GraphedTrainStep(fn, 32, net.params, opt, [net] * listed) if listed else None
        log = []
        for _ in range(4):
            o = torch.nn.functional.normalize(torch.randn((32, 3), generator=g, device=gpu), dim=1) * 4
            t = torch.rand((32, 3), generator=g, device=gpu)
            loss = (step((o, -o / 4), t) if listed else training.train_step(fn, (o, -o / 4), t, net.params, opt))[0]
            log.append(loss.detach().clone())
            assert bool(torch.isfinite(fn((o, -o / 4))[0]).all())    # eager work between the replays
        runs.append([torch.stack(log), net.flat.detach().clone()])
    assert all(torch.equal(x, y) for r in runs[1:] for x, y in zip(r, runs[0]))
