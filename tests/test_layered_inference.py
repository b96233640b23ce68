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
