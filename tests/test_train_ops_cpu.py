"""The training operators without a GPU: what they refuse, the same formulas on CPU tensors, the optimizer's checkpoints, and the
C entry points' checks of their arguments (which come before anything touches a device)."""
import ctypes as C

import pytest
import torch

from alphazero_amd import _lib
from alphazero_amd.network import adamw as A
from alphazero_amd.network.layer_norm import LayerNorm, layer_norm
from tests import train_ops_ref as R

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16, torch.float16])
@pytest.mark.parametrize("shape", [(1,), (3, 5), (2, 3, 4, 361), (0, 7)])
def test_layer_norm_on_the_cpu(shape, dtype):
    torch.manual_seed(0)
    x, w, b, dy = torch.randn(shape).to(dtype), torch.randn(shape[-1]), torch.randn(shape[-1]), torch.randn(shape).to(dtype)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    want, _, r, h = R.norm_forward(x.detach(), w.detach(), b.detach(), 1e-5)
    bounds = R.norm_bounds(x.detach(), w.detach(), b.detach(), dy, 1e-5, dtype, F32)
    for got, ref, tol in zip((y,) + grads, (want,) + R.norm_backward(dy, w.detach(), r, h), bounds):
        # PyTorch's derivative of the formula takes more operations than the kernels' own: eight times their bound
        assert got.shape == ref.shape and bool(((got.double() - ref).abs() <= 8 * tol).all())


def test_layer_norm_refusals():
    x = torch.randn(2, 8)
    for bad, error in [((x.double(),), TypeError), ((x.int(),), TypeError), ((torch.randn(()),), ValueError), ((torch.randn(3, 0),), ValueError),
                       ((x, torch.ones(7)), ValueError), ((x, torch.ones(1, 8)), ValueError), ((x, None, torch.ones(9)), ValueError),
                       ((x, torch.ones(8, dtype=BF16)), TypeError), ((x.bfloat16(), torch.ones(8, dtype=torch.float16)), TypeError),
                       ((x.bfloat16(), torch.ones(8), torch.ones(8, dtype=BF16)), TypeError), ((x, None, None, -1.0), ValueError),
                       ((x, None, None, float("nan")), ValueError), ((x.to("meta"),), ValueError)]:
        with pytest.raises(error):
            layer_norm(*bad)
    m = LayerNorm(8)
    assert m.weight.shape == m.bias.shape == (8,) and torch.equal(m(x), layer_norm(x, torch.ones(8), torch.zeros(8)))


def _lists(n=2, bits=32):
    p = [torch.randn(300) for _ in range(n)]
    g = [torch.randn(300) for _ in range(n)]
    if bits == 32:
        return p, g, [torch.zeros(300) for _ in range(n)], [torch.zeros(300) for _ in range(n)]
    return p, g, [torch.zeros(300, dtype=torch.int8) for _ in range(n)], [torch.zeros(300, dtype=torch.uint8) for _ in range(n)]


def test_adamw_step_refusals():
    p, g, m, v = _lists()
    A.adamw_step([], [], [], [], 1)
    for kw in (dict(step=0), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)),
               dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            A.adamw_step(p, g, m, v, **dict(dict(step=1), **kw))
    with pytest.raises(TypeError):
        A.adamw_step(p, g, m, v, 1, lr=torch.tensor(1e-3))
    with pytest.raises(ValueError):
        A.adamw_step(p, g[:1], m, v, 1)
    with pytest.raises(ValueError):
        A.adamw_step(p, [g[0], g[1][:299]], m, v, 1)
    with pytest.raises(ValueError):
        A.adamw_step(p, [g[0], g[1].view(30, 10)], m, v, 1)
    with pytest.raises(TypeError):
        A.adamw_step(p, [g[0], g[1].bfloat16()], m, v, 1)
    with pytest.raises(TypeError):
        A.adamw_step(p, g, [t.bfloat16() for t in m], v, 1)
    with pytest.raises(TypeError):
        A.adamw_step([t.double() for t in p], [t.double() for t in g], m, v, 1)
    with pytest.raises(ValueError):
        A.adamw_step([torch.randn(600)[::2]], g[:1], m[:1], v[:1], 1)          # not dense
    with pytest.raises(ValueError):
        A.adamw_step([torch.randn(20, 15).t()], [torch.randn(15, 20)], [torch.zeros(15, 20)], [torch.zeros(15, 20)], 1)   # other orders in memory
    p8, g8, m8, v8 = _lists(bits=8)
    scales = [torch.zeros(2), torch.zeros(2)]
    A.adamw_step(p8, g8, m8, v8, 1, exp_avg_scales=scales, exp_avg_sq_scales=[s.clone() for s in scales])
    with pytest.raises(ValueError):
        A.adamw_step(p8, g8, m8, v8, 1, exp_avg_scales=scales)
    with pytest.raises(ValueError):
        A.adamw_step(p8, g8, m8, v8, 1, exp_avg_scales=[torch.zeros(1)] * 2, exp_avg_sq_scales=scales)
    with pytest.raises(TypeError):
        A.adamw_step(p8, g8, m, v, 1, exp_avg_scales=scales, exp_avg_sq_scales=scales)
    with pytest.raises(TypeError):
        A.adamw_step(p8, g8, m8, v8, 1)
    with pytest.raises(ValueError):
        A.adamw_step([torch.randn(3, device="meta")], [torch.randn(3, device="meta")], [torch.zeros(3, device="meta")], [torch.zeros(3, device="meta")], 1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_step_on_the_cpu(dtype, bits):
    torch.manual_seed(1)
    p, g = torch.randn(1000).to(dtype), torch.randn(1000).to(dtype)
    m, v, more = torch.randn(1000) * 0.3, torch.rand(1000) + 0.5, {}
    if bits == 8:
        (m, ms), (v, vs) = A.quantize_state(m, True), A.quantize_state(v, False)
        more = dict(exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    m0, v0 = (R.values(m, ms), R.values(v, vs)) if bits == 8 else (m.clone(), v.clone())
    p2, m2, v2, tp, tm, tv = R.adamw(p, g, m0, v0, 5, 1e-2, 0.9, 0.999, 1e-8, 0.1)
    A.adamw_step([p], [g], [m], [v], 5, lr=1e-2, weight_decay=0.1, **more)
    assert bool(((p.double() - p2).abs() <= tp + R.half_step(dtype) * (p2.abs() + tp)).all())
    if bits == 8:
        for codes, scales, new, signed in ((m, ms, m2, True), (v, vs, v2, False)):
            c, s = R.codes_of(new, signed)
            assert torch.equal(codes, c) and torch.equal(scales, s)
    else:
        assert bool(((m.double() - m2).abs() <= tm).all()) and bool(((v.double() - v2).abs() <= tv).all())


def test_codes_are_the_nearest_and_read_back_as_themselves():
    torch.manual_seed(2)
    for signed in (True, False):
        x = torch.randn(3000) * 10.0 ** (-6 * torch.rand(3000))
        x = x if signed else x.abs()
        codes, scales = A.quantize_state(x, signed)
        c, s = R.codes_of(x.double(), signed)
        assert torch.equal(codes, c) and torch.equal(scales, s)
        g = (torch.randint(1, 257, (3000,)) * 2.0 ** torch.randint(-9, 1, (3000,)))
        g = g if signed else g * g                  # few bits: some lie on a border between two codes
        assert torch.equal(A.quantize_state(g, signed)[0], R.codes_of(g.double(), signed)[0])
        back = A.dequantize_state(codes, scales)
        again, _ = A.quantize_state(back, signed)
        assert torch.equal(again, codes) and back.dtype == F32
        if not signed:
            assert bool((back[x > 0] > 0).all())         # never rounded away
    with pytest.raises(TypeError):
        A.dequantize_state(codes.int(), scales)
    with pytest.raises(ValueError):
        A.dequantize_state(codes, scales[:-1])
    with pytest.raises(ValueError):
        A.quantize_state(x[::2], False)
    x[300] = float("nan")
    back = A.dequantize_state(*A.quantize_state(x, False))
    assert bool(back[256:512].isnan().all()) and bool(back[:256].isfinite().all()) and bool(back[512:].isfinite().all())
    assert A.quantize_state(torch.zeros(0), True)[1].numel() == 0


def test_optimizer_is_adamw():
    """Against PyTorch's own over ten steps, in float64 there: both round each step's parameters in float32 here."""
    torch.manual_seed(3)
    w = [torch.randn(20, 300), torch.randn(7)]
    mine, ref = [t.clone().requires_grad_() for t in w], [t.double().requires_grad_() for t in w]
    a, b = A.AdamW(mine, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.1)
    for _ in range(10):
        for p, q in zip(mine, ref):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.double()
        a.step()
        b.step()
    for p, q in zip(mine, ref):
        assert float((p.detach().double() - q.detach()).abs().max()) <= 10 * (4 * R.U32 * 5 + 40 * R.U32 * 1e-2)
    assert a.step(lambda: torch.tensor(2.0)) == 2.0


def test_optimizer_refusals():
    p = torch.randn(300, requires_grad=True)
    for kw in (dict(lr=-1.0), dict(state_bits=16), dict(betas=(0.9, 1.5))):
        with pytest.raises(ValueError):
            A.AdamW([p], **kw)
    with pytest.raises(TypeError):
        A.AdamW([torch.randn(3, dtype=torch.float64, requires_grad=True)])
    with pytest.raises(ValueError):
        A.AdamW([torch.nn.Parameter(torch.randn(6)[::2])])
    opt = A.AdamW([p])
    with pytest.raises(TypeError):
        opt.add_param_group({"params": [torch.randn(3, dtype=torch.float64, requires_grad=True)]})
    assert len(opt.param_groups) == 1
    sgd = torch.optim.SGD([p], lr=0.1, momentum=0.9)
    p.grad = torch.ones_like(p)
    sgd.step()
    with pytest.raises(ValueError, match="AdamW"):
        opt.load_state_dict(sgd.state_dict())
    q = [torch.randn(300, requires_grad=True), torch.randn(10, 30, requires_grad=True)]
    for t in q:
        t.grad = torch.ones_like(t)
    other, twin = A.AdamW(q, lr=0.5), A.AdamW([torch.randn(300, requires_grad=True), torch.randn(300, requires_grad=True)])
    twin_p = twin.param_groups[0]["params"]
    for t in twin_p:
        t.grad = torch.ones_like(t)
    other.step()
    twin.step()
    twin.step()
    with pytest.raises(ValueError, match="shape"):
        other.load_state_dict(twin.state_dict())
    assert other.param_groups[0]["lr"] == 0.5 and [other.state[t]["step"] for t in q] == [1, 1]     # nothing was changed
    opt.step()
    with pytest.raises(ValueError, match="groups"):
        other.load_state_dict(opt.state_dict())
    theirs = torch.optim.AdamW(twin_p, lr=0.25)
    theirs.step()
    twin.load_state_dict(theirs.state_dict())        # PyTorch's own AdamW has the same state
    assert twin.param_groups[0]["lr"] == 0.25 and twin.state[twin_p[0]]["step"] == 1
    assert torch.equal(twin.state[twin_p[0]]["exp_avg"], theirs.state[twin_p[0]]["exp_avg"])
    twin.step()


def test_optimizer_copies():
    import copy
    import pickle
    torch.manual_seed(6)
    p = torch.randn(5000, requires_grad=True)
    opt = A.AdamW([p], state_bits=8, min_8bit_size=100)
    p.grad = torch.randn_like(p)
    opt.step()
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.state_bits == 8 and other.min_8bit_size == 100
        q, = other.param_groups[0]["params"]
        q.grad = p.grad.clone()
        other.step()
        assert other.state[q]["step"] == 2 and "exp_avg_scale" in other.state[q]
        last = q.detach().clone()
    opt.step()
    assert torch.equal(p.detach(), last)


@pytest.mark.parametrize("first,second", [(32, 32), (8, 8), (32, 8), (8, 32)])
def test_optimizer_checkpoints(first, second, tmp_path):
    """A checkpoint goes through a file and into an optimizer with either kind of state, whose next step is then the same (same
    kind) or that of the converted state."""
    torch.manual_seed(4)
    shapes = [(300, 20), (5,), (16, 40, 3, 3)]
    w = [torch.randn(s) for s in shapes]
    w[2] = w[2].contiguous(memory_format=torch.channels_last)

    def fresh(bits, values):
        ps = [t.clone(memory_format=torch.preserve_format).requires_grad_() for t in values]
        return ps, A.AdamW(ps, lr=1e-2, state_bits=bits)
    ps, opt = fresh(first, w)
    for _ in range(3):
        for p in ps:
            p.grad = torch.randn_like(p)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt")
    qs, opt2 = fresh(second, [p.detach() for p in ps])
    opt2.load_state_dict(torch.load(tmp_path / "opt", weights_only=True))
    for p, q in zip(ps, qs):
        a, b = opt.state[p], opt2.state[q]
        assert b["step"] == 3 and ("exp_avg_scale" in b) == (second == 8 and q.numel() >= 4096)
        assert b["exp_avg"].stride() == q.stride()
        values = [A.dequantize_state(s["exp_avg"], s["exp_avg_scale"]) if "exp_avg_scale" in s else s["exp_avg"] for s in (a, b)]
        if ("exp_avg_scale" in a) == ("exp_avg_scale" in b) or "exp_avg_scale" in a:
            assert torch.equal(*values)
        else:   # to 8 bits: half a code at the top of a block is (1 / 127) of its largest value, less below
            assert float((values[0] - values[1]).abs().max()) <= float(a["exp_avg"].abs().max()) / 127
    if first == second:
        for p, q in zip(ps, qs):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        opt.step()
        opt2.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_checkpoint_of_codes_in_another_memory_order():
    torch.manual_seed(5)
    a = torch.randn(16, 40, 3, 3).contiguous(memory_format=torch.channels_last).requires_grad_()
    b = a.detach().contiguous().requires_grad_()
    one, two = A.AdamW([a], state_bits=8), A.AdamW([b], state_bits=8)
    a.grad = torch.randn_like(a)
    one.step()
    two.load_state_dict(one.state_dict())
    x = A.dequantize_state(one.state[a]["exp_avg"], one.state[a]["exp_avg_scale"])
    y = A.dequantize_state(two.state[b]["exp_avg"], two.state[b]["exp_avg_scale"])
    assert y.is_contiguous() and float((x - y).abs().max()) <= float(x.abs().max()) / 127


def test_c_entry_points_check_their_arguments():
    L = _lib.lib()
    err = lambda: L.az_last_error(None)  # noqa: E731
    fwd = lambda **k: L.az_layer_norm_fwd_dev(*dict(dict(device=0, stream=None, type=0, affine=0, rows=2, cols=4, eps=1e-5, x=4096, xs=4, w=None, b=None,  # noqa: E731
                                                         y=8192, ys=4, mean=None, rstd=None, space=None, n=0), **k).values())
    for bad in (dict(type=7), dict(affine=1), dict(affine=5), dict(rows=-1), dict(cols=0), dict(cols=1 << 26), dict(rows=1 << 49), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(y=None),
                dict(xs=-4), dict(ys=3), dict(mean=4096)):
        assert fwd(**bad) == _lib.ERR_ARG and b"layer norm" in err(), bad
    assert fwd(rows=0) == 0
    assert L.az_layer_norm_fwd_workspace(0, 2, 8192) == 0 and L.az_layer_norm_fwd_workspace(0, 300, 100000) == 0
    assert L.az_layer_norm_fwd_workspace(0, 3, 20000) == 18 and L.az_layer_norm_fwd_workspace(9, 3, 20000) == 0
    for bad in (dict(n=17), dict(space=4100), dict(space=None)):
        assert fwd(**dict(dict(rows=3, cols=20000, xs=20000, ys=20000, space=4096, n=18), **bad)) == _lib.ERR_ARG and b"workspace" in err()
    bwd = lambda **k: L.az_layer_norm_bwd_dev(*dict(dict(device=0, stream=None, type=0, affine=0, rows=2, cols=4, dy=4096, dys=4, x=4096, xs=4, w=None, mean=4096,  # noqa: E731
                                                         rstd=4096, dx=8192, dxs=4, dw=4096, db=None, space=4096, n=16), **k).values())
    assert L.az_layer_norm_bwd_workspace(0, 2, 4) == 8 and not any(L.az_layer_norm_bwd_workspace(*x) for x in ((0, 0, 4), (0, -1, 4), (9, 2, 4)))
    for bad in (dict(type=3), dict(dy=None), dict(x=None), dict(mean=None), dict(n=7), dict(space=None), dict(space=4100), dict(dxs=3), dict(dys=-1)):
        assert bwd(**bad) == _lib.ERR_ARG and b"layer norm" in err(), bad
    assert bwd(dx=None, dw=None) == 0

    def ptrs(*x):
        return (C.c_void_p * len(x))(*x)

    def step(p=(4096, 8192), g=(12288, 16384), m=(20480, 24576), v=(28672, 32768), ms=None, vs=None, n=(10, 10), type=0, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0,
             t=1, count=2):
        return L.az_adamw_step_dev(0, None, count, ptrs(*p), ptrs(*g), ptrs(*m), ptrs(*v), ptrs(*ms) if ms else None, ptrs(*vs) if vs else None,
                                   (C.c_int64 * 2)(*n), type, lr, b1, b2, eps, wd, t)
    for bad in (dict(count=-1), dict(type=9), dict(lr=-1.0), dict(b1=1.0), dict(b2=-0.1), dict(eps=float("nan")), dict(wd=-1.0), dict(t=0), dict(n=(-1, 10)), dict(n=(10, 1 << 36)),
                dict(p=(None, 8192)), dict(g=(12288, None)), dict(ms=(36864, 40960)), dict(ms=(36864, None), vs=(45056, 49152))):
        assert step(**bad) == _lib.ERR_ARG and b"adamw" in err(), bad
    for shared in (dict(p=(4096, 4100)), dict(m=(4096, 24576)), dict(v=(20480, 32768)), dict(g=(4100, 16384)), dict(g=(20500, 16384)),
                   dict(ms=(36864, 36864), vs=(45056, 49152))):
        assert step(**shared) == _lib.ERR_ARG and b"share memory" in err(), shared
    assert step(n=(0, 0)) == 0 and step(count=0) == 0
    assert L.az_dequantize_state_dev(0, None, None, 4096, 4, 1, 4096) == _lib.ERR_ARG and L.az_dequantize_state_dev(0, None, 4096, 4096, -1, 1, 4096) == _lib.ERR_ARG
    assert L.az_dequantize_state_dev(0, None, None, None, 0, 1, None) == 0
