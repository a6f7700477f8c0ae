"""Layer norm and the AdamW step on the GPU against their formulas in 64 bits (tests/train_ops_ref.py), at the sizes, types,
strides and values where they can go wrong."""
import numpy as np
import pytest
import torch

from alphazero_amd.engine import EngineError
from alphazero_amd.network import adamw as A
from alphazero_amd.network.layer_norm import LayerNorm, layer_norm
from tests import train_ops_ref as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inside(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), "%s: %.3g of the bound, at most 1 allowed" % (what, float((off / tol.expand_as(off)).max()))


def _norm_case(rows, cols, dtype, affine, seed, weight=True, bias=True, offset=1.0):
    g = _gen(seed)
    x = (torch.randn(rows, cols, generator=g, device=DEV) + offset * torch.randn(rows, 1, generator=g, device=DEV)).to(dtype)
    w = (1.0 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(affine) if weight else None
    b = (0.3 * torch.randn(cols, generator=g, device=DEV)).to(affine) if bias else None
    dy = torch.randn(rows, cols, generator=g, device=DEV).to(dtype)
    return x, w, b, dy


def _check_norm(x, w, b, dy, eps=1e-5):
    dtype = x.dtype
    affine = (w if w is not None else b).dtype if w is not None or b is not None else F32
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)            # with or without a graph
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    ry, _, r, h = R.norm_forward(x, w, b, eps)
    rdx, rdw, rdb = R.norm_backward(dy, w, r, h)
    ty, tx, tw, tb = R.norm_bounds(x, w, b, dy, eps, dtype, affine)
    _inside(y, ry, ty, "y")
    _inside(grads[0], rdx, tx, "dx")
    k = 1
    if w is not None:
        _inside(grads[k], rdw, tw, "dweight")
        k += 1
    if b is not None:
        _inside(grads[k], rdb, tb, "dbias")


COLS = [1, 2, 3, 4, 5, 30, 63, 64, 65, 128, 255, 256, 257, 361, 511, 512, 513, 722, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192,
        8193, 10001, 16383, 16384, 16385, 33000]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype,affine", [(F32, F32), (BF16, F32), (F16, F16)])
def test_norm_every_width(cols, dtype, affine):
    for rows in (1, 7):
        _check_norm(*_norm_case(rows, cols, dtype, affine, seed=cols + rows))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 15, 16, 17, 361, 4095, 4097, 20011])
@pytest.mark.parametrize("cols,dtype,affine", [(30, F32, F32), (256, BF16, BF16), (361, F32, F32), (1500, F16, F32)])
def test_norm_every_number_of_rows(rows, cols, dtype, affine):
    _check_norm(*_norm_case(rows, cols, dtype, affine, seed=rows))


@pytest.mark.parametrize("rows,cols", [(3, 8193), (255, 8200), (256, 8200), (257, 12345), (3, 300000), (1, 1000001), (100, 24576), (2, 16384), (2, 16385),
                                       (2, 16387), (2, 16388), (2, 16391), (2, 16392), (255, 16392), (256, 16400), (300, 20000), (2000, 16384)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_wide_rows_in_chunks(rows, cols, dtype):
    """Rows too wide for a workgroup, few of them (in chunks) and many."""
    _check_norm(*_norm_case(rows, cols, dtype, F32, seed=rows))


@pytest.mark.parametrize("cols", range(1, 41))
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_narrow_rows(cols, dtype):
    for rows in (1, 63, 64, 65, 5000):
        _check_norm(*_norm_case(rows, cols, dtype, F32, seed=cols))


@pytest.mark.parametrize("cols", [20, 256, 3000, 9000, 20000])
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_norm_without_weight_or_bias(cols, weight, bias):
    _check_norm(*_norm_case(33, cols, F32, F32, seed=3, weight=weight, bias=bias))


@pytest.mark.parametrize("cols", [20, 256, 3000, 9000, 20000])
def test_norm_gradients_one_at_a_time(cols):
    x, w, b, dy = _norm_case(50, cols, F32, F32, seed=4)
    full = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*full), full, dy)
    for i in range(3):
        part = [t.detach().requires_grad_(k == i) for k, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(layer_norm(*part), [part[i]], dy)
        assert torch.equal(got, want[i])


@pytest.mark.parametrize("cols", [48, 256, 700, 2500, 9000, 20000])
@pytest.mark.parametrize("offset", [100.0, 3000.0])
def test_norm_rows_with_a_mean_far_from_zero(cols, offset):
    _check_norm(*_norm_case(40, cols, F32, F32, seed=5, offset=offset))


@pytest.mark.parametrize("cols", [16, 256, 361, 5000, 9001, 20001])
def test_norm_strides(cols):
    g = _gen(6)
    w, b = 1 + 0.1 * torch.randn(cols, generator=g, device=DEV), torch.randn(cols, generator=g, device=DEV)
    wide = torch.randn(6, 10, cols + 13, generator=g, device=DEV)
    dy = torch.randn(6, 10, cols, generator=g, device=DEV)
    _check_norm(wide[:, :, 5:5 + cols], w, b, dy)                       # rows of a wider buffer, odd start
    _check_norm(wide.transpose(0, 1)[:, :, :cols], w, b, dy.transpose(0, 1))   # leading axes that do not merge
    _check_norm(torch.randn(cols, 9, generator=g, device=DEV).t(), w, b, torch.randn(9, cols, generator=g, device=DEV))   # last axis strided
    _check_norm(torch.randn(cols, generator=g, device=DEV), w, b, dy[0, 0])    # a single row without leading axes
    _check_norm(torch.randn(1, cols, generator=g, device=DEV).expand(7, cols), w, b, dy[0, :7])      # one row read seven times
    _check_norm(torch.randn(7, cols, generator=g, device=DEV), w, b, torch.randn(1, cols, generator=g, device=DEV).expand(7, cols))
    _check_norm(torch.randn(7, cols, generator=g, device=DEV), w, b, torch.ones((), device=DEV).expand(7, cols))    # y.sum()'s gradient
    _check_norm(torch.randn(7, cols, generator=g, device=DEV), torch.randn(2 * cols, generator=g, device=DEV)[::2], b, dy[0, :7])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_norm_odd_addresses(dtype):
    g = _gen(7)
    flat = torch.randn(20 * 361 + 1, generator=g, device=DEV).to(dtype)
    dy = torch.randn(20 * 361 + 1, generator=g, device=DEV).to(dtype)
    wb = torch.randn(2 * 361 + 1, generator=g, device=DEV).to(dtype)
    _check_norm(flat[1:].view(20, 361), wb[1:362], wb[362:], dy[1:].view(20, 361))


def test_norm_channels_of_an_image():
    """The trunk's use: channels last in memory, one row for each point."""
    x = torch.randn(3, 256, 9, 9, generator=_gen(8), device=DEV).contiguous(memory_format=torch.channels_last)
    _check_norm(x.permute(0, 2, 3, 1), torch.ones(256, device=DEV), torch.zeros(256, device=DEV), torch.randn(3, 9, 9, 256, generator=_gen(9), device=DEV))


@pytest.mark.parametrize("cols", [8, 256, 9000, 20000])
def test_norm_without_rows(cols):
    x = torch.empty(0, cols, device=DEV, requires_grad=True)
    w, b = torch.ones(cols, device=DEV, requires_grad=True), torch.zeros(cols, device=DEV, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, cols, device=DEV))
    assert y.shape == dx.shape == (0, cols) and not dw.any() and not db.any()


@pytest.mark.parametrize("cols", [12, 200, 361, 3000, 9000, 20000])
def test_norm_values_that_are_not_finite_stay_in_their_row(cols):
    x, w, b, dy = _norm_case(9, cols, F32, F32, seed=10)
    good = layer_norm(x, w, b)
    bad = x.clone()
    bad[2, 0], bad[5, cols - 1], bad[7, cols // 2] = float("inf"), float("nan"), -float("inf")
    bad.requires_grad_()
    y = layer_norm(bad, w, b)
    keep = [0, 1, 3, 4, 6, 8]
    assert torch.equal(y[keep], good[keep]) and bool(y[[2, 5, 7]].isnan().all())
    dx, = torch.autograd.grad(y, bad, dy)
    ref = x.clone().requires_grad_()
    want, = torch.autograd.grad(layer_norm(ref, w, b), ref, dy)
    assert torch.equal(dx[keep], want[keep]) and bool(dx[[2, 5, 7]].isnan().all())


@pytest.mark.parametrize("cols", [1, 40, 256, 361, 9000])
def test_norm_constant_rows(cols):
    """No spread: y is the bias, dx what eps leaves of it."""
    x = torch.full((5, cols), 7.25, device=DEV)
    w, b = torch.full((cols,), 2.0, device=DEV), torch.arange(cols, device=DEV, dtype=F32)
    assert torch.equal(layer_norm(x, w, b), b.expand(5, cols))
    _check_norm(x, w, b, torch.randn(5, cols, generator=_gen(11), device=DEV))


def test_norm_rows_past_32_bit_offsets():
    stride = (1 << 30) + 8
    buf = torch.zeros(2 * stride + 300, dtype=BF16, device=DEV)
    x = buf.as_strided((3, 300), (stride, 1))
    x.copy_(torch.randn(3, 300, generator=_gen(12), device=DEV))
    _check_norm(x, torch.ones(300, device=DEV), None, torch.randn(3, 300, generator=_gen(13), device=DEV).to(BF16))


def test_norm_results_past_32_bit_offsets():
    """More than 2^32 elements of y and dx, from one row of x and dy that is read over and over."""
    rows, cols = (1 << 19) + 5, 8192
    g = _gen(19)
    x, dy = torch.randn(1, cols, generator=g, device=DEV).to(BF16), torch.randn(1, cols, generator=g, device=DEV).to(BF16)
    w = torch.randn(cols, generator=g, device=DEV)
    one = x.clone().requires_grad_()
    y1 = layer_norm(one, w)
    dx1, = torch.autograd.grad(y1, one, dy)
    many = x.expand(rows, cols).detach().requires_grad_()
    y = layer_norm(many, w)
    pick = [0, 1, (1 << 18) - 1, 1 << 18, rows - 2, rows - 1]
    assert torch.equal(y[pick], y1.expand(6, cols))
    dx, = torch.autograd.grad(y, many, dy.expand(rows, cols))
    assert torch.equal(dx[pick], dx1.expand(6, cols))


def test_norm_same_bits_on_every_call():
    x, w, b, dy = _norm_case(30011, 256, F32, F32, seed=14)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    for _ in range(3):
        again = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_norm_gradient_against_differences():
    """Central differences of the kernel's own forward pass: with step e the formula's error is of order e^2 and the
    rounding of y (half a float32 step of about 2, over 2 e, for about 20 outputs) of order 2e-5."""
    x, w, b, dy = _norm_case(2, 10, F32, F32, seed=15)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    e = 2.0 ** -8
    for t, g in zip(leaves, grads):
        for i in range(t.numel()):
            with torch.no_grad():
                flat, ends = t.view(-1), []
                for s in (e, -e):
                    keep = flat[i].clone()
                    flat[i] += s
                    ends.append(float((layer_norm(*leaves) * dy).double().sum()))
                    flat[i] = keep
            assert abs((ends[0] - ends[1]) / (2 * e) - float(g.view(-1)[i])) < 5e-3


@pytest.mark.parametrize("rows,cols", [(512, 722), (3, 20000), (300, 9000), (300, 17000)])
def test_norm_other_stream_and_capture(rows, cols):
    x, w, b, dy = _norm_case(rows, cols, F32, F32, seed=16)
    want = layer_norm(x, w, b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer_norm(x, w, b)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer_norm(x, w, b)
    for seed in (1, 2, 3):                       # replays see the new input, eager work in between
        x.copy_(_norm_case(rows, cols, F32, F32, seed=seed)[0])
        eager = layer_norm(x, w, b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, eager)


def test_norm_refuses_gradients_in_a_capture():
    x, w, b, _ = _norm_case(4, 64, F32, F32, seed=17)
    w.requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            layer_norm(x, w, b)
    torch.cuda.synchronize()
    assert bool(layer_norm(x, w, b).isfinite().all())       # and the process goes on


def test_norm_refuses_forward_mode():
    import torch.autograd.forward_ad as fw
    x, w, b, dy = _norm_case(4, 64, F32, F32, seed=17)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            layer_norm(fw.make_dual(x, dy), w, b)


def test_norm_refuses_a_second_derivative():
    x, w, b, dy = _norm_case(4, 64, F32, F32, seed=18)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(layer_norm(x, w, b), x, dy, create_graph=True)


def test_norm_two_threads_at_once():
    import threading
    cases = [_norm_case(2000, 361, F32, F32, seed=s) for s in (20, 21)]
    want = [layer_norm(*c[:3]) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                if not torch.equal(layer_norm(*cases[k][:3]), want[k]):
                    bad.append(k)
    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_a_failed_call_leaves_nothing_behind():
    """A device that does not exist is an error of that call only, and the current device stays."""
    from alphazero_amd import _lib
    L, x, y = _lib.lib(), torch.randn(4, 8, device=DEV), torch.empty(4, 8, device=DEV)
    call = lambda device: L.az_layer_norm_fwd_dev(device, None, 0, 0, 4, 8, 1e-5, x.data_ptr(), 8, None, None, y.data_ptr(), 8, None, None, None, 0)  # noqa: E731
    torch.cuda.synchronize()
    assert call(999) == _lib.ERR_HIP and b"device" in L.az_last_error(None)
    assert torch.cuda.current_device() == 0 and call(0) == 0
    torch.cuda.synchronize()
    assert torch.equal(y, layer_norm(x))


# ---- AdamW ----------------------------------------------------------------------------------------------------------------
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


def _adamw_inputs(shapes, dtype, bits, seed, fresh=False):
    """Lists (params, grads, m, v, m scales, v scales) with a history, or without one."""
    g = _gen(seed)
    out = [[], [], [], [], [], []]
    for shape in shapes:
        p = torch.randn(shape, generator=g, device=DEV)
        n = p.numel()
        size = 10.0 ** (-3 * torch.rand((), generator=g, device=DEV))
        grad = (torch.randn(shape, generator=g, device=DEV) * size)
        m = torch.zeros(n, device=DEV) if fresh else torch.randn(n, generator=g, device=DEV) * size * 0.3
        v = torch.zeros(n, device=DEV) if fresh else (0.5 + torch.rand(n, generator=g, device=DEV)) * size ** 2
        if bits == 8:
            (m, ms), (v, vs) = R.codes_of(m.double(), True), R.codes_of(v.double(), False)
            out[4].append(ms)
            out[5].append(vs)
        for k, t in enumerate((p.to(dtype), grad.to(dtype), m.view(shape), v.view(shape))):
            out[k].append(t)
    return out


def _step_all(args, step, **hyper):
    p, g, m, v, ms, vs = args
    A.adamw_step(p, g, m, v, step, **hyper, **(dict(exp_avg_scales=ms, exp_avg_sq_scales=vs) if ms else {}))


def _check_step(args, step, flat=lambda t: t.reshape(-1), **hyper):
    """Runs one step and compares every tensor with the formula."""
    old = [[t.clone() for t in x] for x in args]
    _step_all(args, step, **hyper)
    beta1, beta2 = hyper["betas"]
    for i, p in enumerate(args[0]):
        eight = bool(args[4])
        p0, g0, m0, v0 = (flat(old[k][i]) for k in range(4))
        if eight:
            m0, v0 = R.values(m0, old[4][i]), R.values(v0, old[5][i])
        p2, m2, v2, tp, tm, tv = R.adamw(p0, g0, m0, v0, step, hyper["lr"], beta1, beta2, hyper["eps"], hyper["weight_decay"])
        _inside(flat(p), p2, tp + R.half_step(p.dtype) * (p2.abs() + tp) + R.tiny(p.dtype), "parameter %d" % i)
        if not eight:
            _inside(flat(args[2][i]), m2, tm, "m %d" % i)
            _inside(flat(args[3][i]), v2, tv, "v %d" % i)
            continue
        for k, new, signed in ((2, m2, True), (3, v2, False)):
            codes, scales = R.codes_of(new, signed)
            assert torch.equal(flat(args[k][i]), codes) and torch.equal(args[k + 2][i], scales), "state %d of tensor %d" % (k, i)
            back = A.dequantize_state(args[k][i], args[k + 2][i])
            want = R.values(flat(args[k][i]), scales)
            assert back.shape == args[k][i].shape
            _inside(flat(back), want, 2 * R.U32 * want.abs() + 2.0 ** -149, "values")


SHAPES = [(1,), (2, 3), (), (255,), (256,), (257,), (0, 4), (1023,), (1024,), (1025,), (361, 722), (17, 3, 3, 3), (4096,), (5000,), (2049,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("step,fresh", [(1, True), (2, False), (1000, False), (10 ** 6, False)])
def test_adamw_step(dtype, bits, step, fresh):
    _check_step(_adamw_inputs(SHAPES, dtype, bits, seed=step, fresh=fresh), step, **HYPER)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("hyper", [dict(lr=0.0), dict(weight_decay=0.0), dict(betas=(0.0, 0.0)), dict(betas=(0.0, 0.99)), dict(eps=1.0), dict(eps=1e-12), dict(eps=0.0), dict(lr=1.0, weight_decay=1.0)])
def test_adamw_other_constants(bits, hyper):
    _check_step(_adamw_inputs(SHAPES, F32, bits, seed=5), 7, **dict(HYPER, **hyper))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("betas", [(0.9, 0.0), (0.0, 0.0), (0.0, 0.999)])
def test_adamw_codes_on_a_border(dtype, betas):
    """Without a memory of earlier steps the states of 16-bit gradients are squares and products of few bits, some of which lie
    exactly between two codes."""
    for seed in range(3):
        args = _adamw_inputs([(20000,), (300,)], dtype, 8, seed=seed)
        args[1][1] = (2.0 ** torch.randint(-6, 1, (300,), generator=_gen(seed), device=DEV)).to(dtype)      # g = gmax / 4: half of the root
        _check_step(args, 3, **dict(HYPER, betas=betas))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 55, 56, 57, 63, 64, 65, 112, 113, 128, 129, 300])
def test_adamw_many_tensors(bits, count):
    """More tensors than one launch's table holds, of every size, empty ones among them."""
    rng = np.random.RandomState(count)
    shapes = [(int(n),) for n in rng.randint(0, 3000, count)]
    _check_step(_adamw_inputs(shapes, F32, bits, seed=count), 3, **HYPER)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [(1 << 20) - 1, (1 << 20) + 1, 5 * (1 << 20) + 257])
def test_adamw_large_tensors(bits, n):
    _check_step(_adamw_inputs([(n,), (3,)], BF16, bits, seed=n), 3, **HYPER)


@pytest.mark.parametrize("bits,dtype,n", [(32, F32, 9586981), (32, BF16, 12201612), (8, F32, 16777216), (8, F32, 16777217), (8, BF16, 26843546)])
def test_adamw_steps_past_the_caches(bits, dtype, n):
    """Around and beyond 256 MB of weights, gradients and states, from where the step streams; small tensors beside the large
    one, so that chunks end inside a tensor."""
    _check_step(_adamw_inputs([(5,), (n,), (4097,), (1023,)], dtype, bits, seed=n), 3, **HYPER)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_past_32_bit_offsets(bits):
    """A tensor of more than 2^31 elements (all zeros but for three stretches), the stretches compared with the formula."""
    n, length = (1 << 31) + 4097, 5000
    at = [0, ((1 << 30) // 256 - 3) * 256, ((n - length) // 256) * 256]
    small = _adamw_inputs([(length,), (length,), (n - at[2],)], BF16, bits, seed=44)
    types = (torch.int8, torch.uint8) if bits == 8 else (F32, F32)
    args = [[torch.zeros(n, dtype=t, device=DEV)] for t in (BF16, BF16) + types] + [[], []]
    if bits == 8:
        args[4], args[5] = [torch.zeros(-(-n // 256), device=DEV)], [torch.zeros(-(-n // 256), device=DEV)]
    for k in range(6 if bits == 8 else 4):
        for a, t in zip(at, small[k]):
            a = a // 256 if k > 3 else a
            args[k][0][a:a + t.numel()] = t
    _step_all(args, 9, **HYPER)
    _step_all(small, 9, **HYPER)      # small tensors are compared with the formula elsewhere
    for k in range(6 if bits == 8 else 4):
        for a, t in zip(at, small[k]):
            a = a // 256 if k > 3 else a
            assert torch.equal(args[k][0][a:a + t.numel()], t)
        gap = slice((1 << 20) // (256 if k > 3 else 1), (1 << 22) // (256 if k > 3 else 1))     # between the stretches
        assert not args[k][0][gap].any()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_tensors_packed_without_gaps_leave_their_neighbours_alone(dtype, bits):
    """Views into flat buffers, each starting where the last one ended, with a guard after every tensor that must stay."""
    sizes = [1, 3, 257, 1000, 511, 4097, 7]
    g = _gen(30)
    total = sum(sizes) + len(sizes)
    flat = [torch.randn(total, generator=g, device=DEV).to(dtype) for _ in range(2)]
    state = [torch.randint(-100, 100, (total,), generator=g, device=DEV).to(torch.int8), torch.randint(1, 255, (total,), generator=g, device=DEV).to(torch.uint8)] \
        if bits == 8 else [torch.randn(total, generator=g, device=DEV), torch.rand(total, generator=g, device=DEV)]
    buffers = flat + state
    starts = np.cumsum([0] + [n + 1 for n in sizes])[:-1]
    args = [[b[a:a + n] for a, n in zip(starts, sizes)] for b in buffers] + [[], []]
    if bits == 8:
        args[4] = [torch.rand(-(-n // 256), generator=g, device=DEV) for n in sizes]
        args[5] = [torch.rand(-(-n // 256), generator=g, device=DEV) for n in sizes]
    guards = torch.as_tensor([int(a) + n for a, n in zip(starts, sizes)], device=DEV)
    before = [b[guards].clone() for b in buffers]
    _check_step(args, 4, **HYPER)
    for b, want in zip(buffers, before):
        assert torch.equal(b[guards], want)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_channels_last_tensors(bits):
    def order(t):
        return t.permute(0, 2, 3, 1).reshape(-1) if t.dim() == 4 else t.reshape(-1)
    args = _adamw_inputs([(8, 17, 3, 3), (33, 5, 7, 3)], F32, bits, seed=31)
    for k in range(4):
        args[k] = [t.contiguous(memory_format=torch.channels_last) for t in args[k]]
    _check_step(args, 2, flat=order, **HYPER)


def test_adamw_zero_gradients_and_no_history():
    for bits in (32, 8):
        args = _adamw_inputs([(300,), (5000,)], F32, bits, seed=32, fresh=True)
        args[1] = [torch.zeros_like(t) for t in args[1]]
        before = [t.clone() for t in args[0]]
        _step_all(args, 1, **dict(HYPER, weight_decay=0.0))
        assert all(torch.equal(p, q) for p, q in zip(args[0], before)) and not any(t.any() for k in (2, 3, 4, 5) for t in args[k])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-8, 1e-20, 1e-30])
@pytest.mark.parametrize("size", [1e-12, 1e-16, 3e-17, 1e-18])
def test_adamw_squares_near_the_smallest_numbers(bits, eps, size):
    """v from 1e-24 down into the subnormal numbers (below 1.2e-38), with an eps beside which its root counts or does not; blocks
    that hold values of very different size.  A subnormal v is itself only right to half of its last place, 2^-150."""
    for mix in (1.0, 1e-3):
        args = _adamw_inputs([(3000,)], F32, bits, seed=45, fresh=True)
        g = torch.randn(3000, generator=_gen(46), device=DEV) * size
        g[::3] *= mix
        args[1] = [g]
        old = args[0][0].clone()
        _step_all(args, 2, **dict(HYPER, eps=eps))
        want, m2, v2, tol, _, _ = R.adamw(old, g, torch.zeros(3000, device=DEV), torch.zeros(3000, device=DEV), 2, HYPER["lr"], 0.9, 0.999, eps, HYPER["weight_decay"])
        root, den = (v2 / (1 - 0.999 ** 2)) ** 0.5, (v2 / (1 - 0.999 ** 2)) ** 0.5 + eps
        lost = 1.0 - ((v2 - 2.0 ** -149).clamp(min=0.0) / v2.clamp(min=1e-300)) ** 0.5        # of the root, relative
        tol = tol + (old.double() - want).abs() * (root * lost / (den - root * lost).clamp(min=1e-300)).clamp(max=1e6)
        seen = v2 > 2.0 ** -148
        assert bool(((args[0][0].double() - want).abs() <= tol)[seen].all())
        if bits == 8:
            for k, new, signed in ((2, m2, True), (3, v2, False)):
                codes, scales = R.codes_of(new, signed)
                assert torch.equal(args[k][0], codes) and torch.equal(args[k + 2][0], scales)


def test_adamw_tiny_values():
    """Gradients whose squares leave float32 and blocks whose scale is subnormal."""
    for bits in (32, 8):
        for size in (1e-25, 1e-40):
            args = _adamw_inputs([(700,)], F32, bits, seed=33, fresh=True)
            args[1] = [t * size for t in args[1]]
            _step_all(args, 1, **HYPER)
            assert all(bool(t.isfinite().all()) for t in args[0])
            if bits == 8:
                for k, signed in ((2, True), (3, False)):
                    g = args[1][0].double()
                    codes, scales = R.codes_of(0.1 * g if signed else (1 - 0.999) * g * g, signed)
                    # (the factor 1 - 0.9 in 64 bits is not 0.1 to the last bit: scales may differ by a step)
                    assert torch.allclose(args[k + 2][0], scales, rtol=2.0 ** -22, atol=2.0 ** -149)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_adamw_gradients_that_are_not_finite(bad):
    """32 bits: the element alone.  8 bits: its block's state reads back as NaN, the other blocks and the weights of its
    neighbours are untouched by it."""
    for bits in (32, 8):
        args, clean = (_adamw_inputs([(1000,)], F32, bits, seed=34) for _ in range(2))
        args[1][0][300] = bad
        _step_all(args, 3, **HYPER)
        _step_all(clean, 3, **HYPER)
        other = torch.arange(1000, device=DEV) != 300
        assert torch.equal(args[0][0][other], clean[0][0][other]) and bool(args[0][0][300].isnan())
        if bits == 32:
            assert torch.equal(args[2][0][other], clean[2][0][other]) and not bool(args[2][0][300].isfinite())
            continue
        for k in (2, 3):
            got, want = A.dequantize_state(args[k][0], args[k + 2][0]), A.dequantize_state(clean[k][0], clean[k + 2][0])
            block = (torch.arange(1000, device=DEV) // 256) == 1
            assert bool(got[block].isnan().all()) and torch.equal(got[~block], want[~block])


def test_adamw_refusals():
    p, g, m, v, _, _ = _adamw_inputs([(100,), (50,)], F32, 32, seed=35)
    flat = torch.zeros(150, device=DEV)
    with pytest.raises(EngineError, match="share memory"):
        A.adamw_step([flat[:100], flat[80:130]], g, m, v, 1)
    with pytest.raises(EngineError, match="share memory"):
        A.adamw_step([p[0], p[0]], [g[0], g[0]], [m[0], m[0]], [v[0], v[0]], 1)
    with pytest.raises(EngineError, match="share memory"):
        A.adamw_step(p, [m[0], g[1]], m, v, 1)            # a gradient that the step writes
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            A.adamw_step(p, g, m, v, 1)
    torch.cuda.synchronize()
    A.adamw_step(p, [g[0], g[0][:50]], m, v, 1)           # two gradients may be the same memory
    with pytest.raises(ValueError, match="not on"):
        A.adamw_step(p, [g[0], g[1].cpu()], m, v, 1)


def test_adamw_refused_capture_leaves_no_state():
    """A first step that is refused in a capture has made no state in the graph's memory; the next one is right."""
    w = [torch.randn(5000, generator=_gen(k), device=DEV).requires_grad_() for k in (1, 1)]
    a, b = A.AdamW(w[:1], state_bits=8), A.AdamW(w[1:], state_bits=8)
    for t in w:
        t.grad = torch.randn(5000, generator=_gen(2), device=DEV)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            a.step()
    torch.cuda.synchronize()
    assert not a.state
    del graph
    a.step()
    b.step()
    assert torch.equal(w[0].detach(), w[1].detach())


def test_adamw_tells_autograd():
    w = torch.randn(300, device=DEV, requires_grad=True)
    y = (w * w).sum()
    w.grad = torch.ones_like(w)
    opt = A.AdamW([w])
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_adamw_other_stream():
    a, b = _adamw_inputs(SHAPES, F32, 8, seed=36), _adamw_inputs(SHAPES, F32, 8, seed=36)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for t in (1, 2, 3):
            _step_all(a, t, **HYPER)
    for t in (1, 2, 3):
        _step_all(b, t, **HYPER)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for p, q in zip(a, b) for x, y in zip(p, q))


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_on_the_gpu_is_the_optimizer_on_the_cpu(bits):
    """Five steps of the class on both devices; a gradient that is missing, one laid out otherwise, one parameter group with
    constants of its own.  The CPU path is held to the formula in tests/test_train_ops_cpu.py.  Both sides round in float32,
    so parameters agree to a few steps of the sum of their updates, and in 8 bits to that plus what a code that fell on
    the other side of a border can do to later steps (none does for these seeds: the codes are compared)."""
    torch.manual_seed(37)
    shapes = [(300, 20), (5,), (16, 8, 3, 3), (5000,)]
    start = [torch.randn(s) for s in shapes]
    opts, params = [], []
    for dev in ("cpu", DEV):
        ps = [t.clone().to(dev).requires_grad_() for t in start]
        ps[2].data = ps[2].data.contiguous(memory_format=torch.channels_last)
        opts.append(A.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 3e-3, "weight_decay": 0.0}], lr=1e-3, state_bits=bits))
        params.append(ps)
    for k in range(5):
        grads = [torch.randn(s) for s in shapes]
        for ps, opt in zip(params, opts):
            for i, (p, g) in enumerate(zip(ps, grads)):
                p.grad = None if (k, i) == (1, 3) else g.to(p.device)
            opt.step()
    for p, q, s in zip(*params, shapes):
        assert q.is_contiguous(memory_format=torch.channels_last) if len(s) == 4 else True
        assert float((p.detach() - q.detach().cpu()).abs().max()) <= 5 * (8 * R.U32 * 5 + 32 * R.U32 * 3e-3)
    for p, q in zip(*params):
        a, b = opts[0].state[p], opts[1].state[q]
        assert a["step"] == b["step"]
        if "exp_avg_scale" in a:
            assert torch.equal(a["exp_avg"], b["exp_avg"].cpu()) and torch.equal(a["exp_avg_sq"], b["exp_avg_sq"].cpu())


def test_layer_norm_module_trains_with_the_optimizer():
    """A step through both operators as a training loop uses them, against the same step in 64 bits."""
    torch.manual_seed(38)
    net = torch.nn.Sequential(torch.nn.Linear(30, 361), LayerNorm(361), torch.nn.ReLU(), torch.nn.Linear(361, 5)).to(DEV)
    ref = torch.nn.Sequential(torch.nn.Linear(30, 361), torch.nn.LayerNorm(361), torch.nn.ReLU(), torch.nn.Linear(361, 5)).double()
    ref.load_state_dict({k: v.double().cpu() for k, v in net.state_dict().items()})
    opt = A.AdamW(net.parameters(), lr=1e-3, weight_decay=0.1)
    x, t = torch.randn(64, 30), torch.randn(64, 5)
    loss = ((net(x.to(DEV)) - t.to(DEV)) ** 2).mean()
    loss.backward()
    ((ref(x.double()) - t.double()) ** 2).mean().backward()
    for (name, p), q in zip(net.named_parameters(), ref.parameters()):
        # sums of 64 * 361 float32 products at most, each off by a few half steps: 1e-4 of the largest gradient
        assert float((p.grad.cpu().double() - q.grad).abs().max()) <= 1e-4 * float(q.grad.abs().max()) + 1e-7, name
    before = [p.detach().clone() for p in net.parameters()]
    opt.step()
    for p, b in zip(net.parameters(), before):
        g = p.grad.double()
        want = b.double() * (1 - 1e-4) - 1e-3 * g / (g.abs() + 1e-8)     # first step: m / sqrt(v) is the gradient's sign
        assert float((p.detach().double() - want).abs().max()) <= 8 * R.U32 * (float(b.abs().max()) + 1e-3) + 1e-3 * 32 * R.U32
