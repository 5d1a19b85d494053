"""AdamW steps at the edges of what there is to step."""

import pytest
import torch

from triton_pesq_b200 import AdamWCuda, adamw_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("units", [0, 1])
def test_a_step_without_values_counts(cuda_device, bits, units):
    def state():
        kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
        m, v = (torch.zeros(256 * units, device=cuda_device).to(kind) for _ in range(2))
        scales = torch.zeros(2, units, device=cuda_device) if bits == 8 else None
        return m, v, torch.tensor([4, 0], device=cuda_device), scales

    empty = torch.zeros(0, device=cuda_device)
    for params in ([], [empty], [empty, torch.zeros(3, 0, device=cuda_device)]):
        m, v, step, scales = state()
        adamw_step(params, [torch.zeros_like(p) for p in params], m, v, step, scales=scales)
        assert step.tolist() == [5, 0]
        adamw_step(params, [torch.zeros_like(p) for p in params], m, v, step, scales=scales,
                   grad_scale=torch.full((1,), float("inf"), device=cuda_device))
        assert step.tolist() == [5, 0]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_group_of_empty_parameters_steps(cuda_device, bits):
    empty, one = torch.nn.Parameter(torch.zeros(0, device=cuda_device)), torch.nn.Parameter(torch.ones(3, device=cuda_device))
    opt = AdamWCuda([{"params": [empty]}, {"params": [one]}], state_bits=bits)
    for n in (1, 2):
        empty.grad, one.grad = torch.zeros_like(empty), torch.ones_like(one)
        opt.step()
        assert opt.state[empty]["step"].tolist() == opt.state[one]["step"].tolist() == [n, 0]


def test_small_gradients_without_eps(cuda_device):
    """Gradients whose squares are below the normal range, eps = 0: the first step moves every value by lr.  The
    second moment, 1e-43, is a multiple of 2**-149, so off by up to 0.7 % and its root by 0.35 %: 0.5 % is allowed."""

    p, g = [torch.zeros(300, device=cuda_device)], [torch.full((300,), 1e-20, device=cuda_device)]
    m, v = torch.zeros(512, device=cuda_device), torch.zeros(512, device=cuda_device)
    adamw_step(p, g, m, v, torch.zeros(2, dtype=torch.int64, device=cuda_device), lr=1.0, eps=0.0, weight_decay=0.0)
    assert float((p[0] + 1).abs().max()) <= 5e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_first_step_is_not_captured(cuda_device, dtype):
    """Its state would be made anew by every replay."""

    w = torch.nn.Parameter(torch.ones(40, device=cuda_device, dtype=dtype))
    w.grad = torch.ones_like(w)
    opt = AdamWCuda([w])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(graph):
            opt.step()
    del graph
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    assert opt.state[w]["step"].tolist() == [4, 0]


def test_layouts_that_are_not_dense_are_refused_at_once(cuda_device):
    weight = torch.nn.Conv2d(3, 4, 3).to(cuda_device, memory_format=torch.channels_last).weight
    for p in (weight, torch.nn.Parameter(torch.ones(6, 4, device=cuda_device).t())):
        with pytest.raises(RuntimeError, match="dense"):
            AdamWCuda([p])
        opt = AdamWCuda([torch.nn.Parameter(torch.ones(2, device=cuda_device))])
        with pytest.raises(RuntimeError, match="dense"):
            opt.add_param_group({"params": [p]})
        assert len(opt.param_groups) == 1
    with pytest.raises(RuntimeError, match="supports"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(2, device=cuda_device).double())]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": (torch.nn.Parameter(torch.ones(n, device=cuda_device)) for n in (1, 2))})
    assert [len(g["params"]) for g in opt.param_groups] == [1, 2]
