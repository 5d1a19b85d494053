"""Which parameters of the example's enhancer are stepped by which optimiser."""

import pytest
import torch

from examples import enhancer
from triton_pesq_b200 import LayerNormCuda


class Stop(Exception):
    pass


@pytest.mark.parametrize("mixer", ["scan", "attention"])
def test_muon_steps_the_blocks_linear_maps_alone(monkeypatch, mixer):
    """The norms' weights [head, channel] are vectors, one for each head: only matrices that a product is made with are
    orthogonalised, and every parameter has one optimiser."""

    given = {}

    class Adam:
        def __init__(self, params, **kw):
            given["adam"] = list(params)

    class Muon:
        def __init__(self, params, **kw):
            given["muon"] = list(params)
            raise Stop

    monkeypatch.setattr(enhancer, "AdamWCuda", Adam)
    monkeypatch.setattr(enhancer, "MuonCuda", Muon)
    model = enhancer.Enhancer(width=32, blocks=2, mixer=mixer)
    with pytest.raises(Stop):
        enhancer.train(model, 1, muon=True)
    linear = [m.weight for b in model.blocks for m in b.modules() if isinstance(m, torch.nn.Linear)]
    assert len(linear) == 4 and {id(p) for p in given["muon"]} == {id(p) for p in linear}
    both = [id(p) for p in (*given["muon"], *given["adam"])]
    assert sorted(both) == sorted(id(p) for p in model.parameters())
    norms = [p for m in model.modules() if isinstance(m, LayerNormCuda) for p in m.parameters()]
    assert len(norms) == (4 if mixer == "attention" else 0) and {id(p) for p in norms} <= {id(p) for p in given["adam"]}
