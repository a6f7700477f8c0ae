"""Tracers do not see inside the training operators: on the GPU they refuse to be traced, where a tracer would keep the result
for one input as a constant.  On the CPU they are PyTorch operations and trace as such."""
import pytest
import torch

from alphazero_amd.network import adamw as A
from alphazero_amd.network.layer_norm import LayerNorm, layer_norm


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_layer_norm_refuses_to_be_traced(grad):
    net = torch.nn.Sequential(torch.nn.Linear(8, 16), LayerNorm(16), torch.nn.Linear(16, 2)).cuda()
    x = torch.randn(3, 8, device="cuda")
    with torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(net, x, check_trace=False)
        assert bool(net(x).isfinite().all())         # and goes on afterwards


@pytest.mark.gpu
def test_layer_norm_refuses_a_graph_of_proxies():
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(3, 8, device="cuda")
    for mode in ("real", "fake", "symbolic"):
        with torch.no_grad(), pytest.raises(RuntimeError):
            make_fx(lambda t: layer_norm(t) + 1, tracing_mode=mode)(x)
    with torch.no_grad():
        assert torch.equal(layer_norm(x), layer_norm(x.clone()))


@pytest.mark.gpu
def test_modes_that_only_watch_are_no_tracers():
    from torch.utils.flop_counter import FlopCounterMode
    x = torch.randn(3, 8, device="cuda")
    want = layer_norm(x)
    with FlopCounterMode(display=False):
        assert torch.equal(layer_norm(x), want)


@pytest.mark.gpu
def test_adamw_and_its_states_refuse_to_be_traced():
    p, g, m, v = (torch.randn(300, device="cuda") for _ in range(4))
    codes, scales = A.quantize_state(torch.randn(300, device="cuda"), True)

    def step(t):
        A.adamw_step([p], [t], [m], [v.abs_()], 1)
        return p * 1.0
    for fn, x in ((step, g), (lambda c: A.dequantize_state(c, scales) * 2.0, codes)):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(fn, x, check_trace=False)


def test_on_the_cpu_a_trace_computes():
    net = torch.nn.Sequential(torch.nn.Linear(8, 16), LayerNorm(16), torch.nn.Linear(16, 2))
    x, other = torch.randn(3, 8), torch.randn(3, 8)
    with torch.no_grad():
        traced = torch.jit.trace(net, x)
        assert torch.allclose(traced(other), net(other), atol=1e-6) and not torch.allclose(traced(other), net(x), atol=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_networks_leave_the_operator_as_it_is(backend):
    """torch.compile breaks its graph at the call and goes on behind it."""
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(8, 16), LayerNorm(16), torch.nn.Linear(16, 2)).cuda()
    compiled = torch.compile(net, backend=backend)
    for k in range(3):
        x = torch.randn(3, 8, device="cuda")
        grads = [torch.autograd.grad(f(x).square().sum(), list(net.parameters())) for f in (net, compiled)]
        assert all(torch.allclose(a, b, rtol=1e-4, atol=1e-5) for a, b in zip(*grads))
