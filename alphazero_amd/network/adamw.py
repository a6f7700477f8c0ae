"""AdamW over all tensors of a network at once, as one HIP kernel (csrc/az_adamw_kernels.h), with its state in 32 or 8 bits.

    m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
    w = w - lr wd w - lr m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps)

It stands beside the momentum SGD of the reference's optimizer (network/main.py:66-88) as `optimizer: adamw` / `adamw8` of
`Network`'s training config.  The weight decay is AdamW's own, applied to the weight and not through the gradient.

8-bit state: blocks of STATE_BLOCK elements, in the order in which they lie in memory, share one float32 scale s, the block's
largest magnitude;  m = s sgn(c) (c / 127)^2 with c int8,  v = s (c / 255)^4 with c uint8 (at least 1 where v > 0);  c is the nearest in
the domain in which codes are evenly spaced, the even one of two that are equally near.  The step
itself uses the new means before they are rounded to codes.  A block that holds an infinity or a NaN reads back as NaN.

Tensors on the GPU go through the kernel, on PyTorch's current stream; tensors on the CPU take the same formulas in PyTorch.
"""
import torch

from .device_ops import TYPES, binding, check, dense, in_memory_order

STATE_BLOCK = 256   # AZ_STATE_BLOCK of include/az_engine.h


def _blocks(n):
    return -(-n // STATE_BLOCK)


def _companded(x, s, power, top):
    """Codes of |x| <= s, x = s (c / top)^power with power 2 or 4: what the roots say, put right by comparing powers at the two
    borders of that code."""
    s, x = s.double(), x.abs()
    root = torch.sqrt(x / torch.where(s > 0, s, torch.ones_like(s)))
    c = ((torch.sqrt(root) if power == 4 else root) * top).round().clamp(max=top)
    scaled, odd = x * (2.0 * top) ** power, c % 2 == 1
    high, low = ((2 * c + 1) ** power) * s, torch.where(c > 0, ((2 * c - 1) ** power) * s, torch.full_like(x, -1.0))
    up, down = (scaled > high) | ((scaled == high) & odd), (scaled < low) | ((scaled == low) & odd)
    return torch.where(s > 0, (c + up.double() - down.double()).clamp(max=top), torch.zeros_like(x))


def quantize_state(values, signed):
    """(codes, scales) of a state held in 32 bits: int8 codes for signed values (m), uint8 for others (v); the codes have the
    shape and the layout of `values` (dense), scales one float32 for every STATE_BLOCK elements in memory order."""
    if not dense(values):
        raise ValueError("a state in 8 bits needs a dense tensor")
    codes = torch.empty_like(values, dtype=torch.int8 if signed else torch.uint8)
    n = values.numel()
    flat = torch.zeros(_blocks(n) * STATE_BLOCK, dtype=torch.float64, device=values.device)
    flat[:n] = in_memory_order(values)
    flat = flat.view(-1, STATE_BLOCK)
    scales = flat.abs().amax(1).float() if n else flat.new_zeros(0, dtype=torch.float32)
    s = scales[:, None]
    fine = torch.isfinite(s) & (s > 0)
    if signed:
        c = _companded(flat, s, 2, 127.0) * flat.sign()
    else:
        c = _companded(flat, s, 4, 255.0)
        c = torch.where(flat > 0, c.clamp(min=1.0), c)
    c = torch.where(fine, c, torch.zeros_like(c))
    in_memory_order(codes).copy_(c.view(-1)[:n])
    return codes, scales


def _values64(codes, scales):
    """The values of codes in memory order, in 64 bits (PyTorch)."""
    c = in_memory_order(codes).double()
    s = scales.double().repeat_interleave(STATE_BLOCK)[:codes.numel()]
    return s * (c * c.abs()) * (1.0 / 16129.0) if codes.dtype == torch.int8 else s * (c * c) ** 2 * (1.0 / 4228250625.0)


def dequantize_state(codes, scales):
    """The float32 values that an 8-bit state stands for, in the shape and layout of `codes`: int8 codes are m, uint8 codes v."""
    out = binding().dequantize_state(codes, scales)
    if out is None:   # on the CPU
        out = torch.empty_like(codes, dtype=torch.float32)
        in_memory_order(out).copy_(_values64(codes, scales))
    return out


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               exp_avg_scales=None, exp_avg_sq_scales=None):
    """One AdamW step, in place, over lists of tensors: params and grads of one type (float32, bfloat16, float16) on one device,
    and the states, in 32 bits (float32) or, with the scales of their blocks given, in 8 (int8 and uint8 codes).  `step` counts
    from 1 and includes this step.  The tensors of one parameter have one shape and lie in memory in one order without gaps
    (contiguous, or all with the same strides).  No two tensors may share memory, and no gradient may share it with what the step
    writes.  The scalars are fixed when the call is made, so it refuses to be captured into a HIP graph, which would replay
    the same step number."""
    if isinstance(lr, torch.Tensor) or isinstance(step, torch.Tensor):
        raise TypeError("lr and step are Python numbers")   # (reading a tensor's would wait for the GPU)
    rc = binding().adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas[0], betas[1], eps, weight_decay, exp_avg_scales, exp_avg_sq_scales)
    check(rc)
    if rc:   # tensors on the CPU
        with torch.no_grad():
            for x in zip(params, grads, exp_avgs, exp_avg_sqs, *([exp_avg_scales, exp_avg_sq_scales] if exp_avg_scales is not None else [])):
                _plain_step(*x[:4], step, lr, betas, eps, weight_decay, *x[4:])


def _plain_step(p, g, m, v, step, lr, betas, eps, weight_decay, m_scale=None, v_scale=None):
    """The step in PyTorch, for tensors on the CPU."""
    beta1, beta2 = betas
    p_, g_, m_, v_ = map(in_memory_order, (p, g, m, v))
    if m_scale is not None:
        g64 = g_.double()
        m64 = _values64(m, m_scale) * beta1 + g64 * (1.0 - beta1)
        v64 = _values64(v, v_scale) * beta2 + g64 * g64 * (1.0 - beta2)
        for value, codes, scale, signed in ((m64, m_, m_scale, True), (v64, v_, v_scale, False)):
            c, s = quantize_state(value, signed)
            codes.copy_(c)
            scale.copy_(s)
        new_m, new_v = m64.float(), v64.float()
    else:
        g32 = g_.float()
        new_m = m_.mul_(beta1).add_(g32 * (1.0 - beta1))
        new_v = v_.mul_(beta2).add_(g32 * g32 * (1.0 - beta2))
    w = p_.float()
    denom = torch.sqrt(new_v) * (1.0 / (1.0 - beta2 ** step) ** 0.5) + eps
    p_.copy_(w - w * (lr * weight_decay) - new_m / denom * (lr / (1.0 - beta1 ** step)))


_CONSTANTS = ("lr", "betas", "eps", "weight_decay")    # of a group (PyTorch adds to self.defaults when a state is set)
_STATE_KEYS = {"step", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"}
# what PyTorch's optimizers of this family keep in their groups beside the constants
_TORCH_KEYS = {"amsgrad", "maximize", "foreach", "capturable", "differentiable", "fused", "decoupled_weight_decay"}


class AdamW(torch.optim.Optimizer):
    """AdamW as a PyTorch optimizer.  state_bits=8 holds the state of every parameter of at least `min_8bit_size` elements in
    8 bits (biases and other small tensors stay in 32).  A checkpoint of either kind loads into the other.

    Parameters are dense tensors of float32, bfloat16 or float16.  A gradient that lies in memory otherwise than its
    parameter is copied first.  Parameters and gradients of one step may not share memory."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, min_8bit_size=4096):
        if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0 and 0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("lr, eps and weight_decay must not be negative, betas must lie in [0, 1)")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self.state_bits, self.min_8bit_size = state_bits, int(min_8bit_size)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def __getstate__(self):   # (what copy and pickle take along)
        return dict(super().__getstate__(), state_bits=self.state_bits, min_8bit_size=self.min_8bit_size)

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            for p in self.param_groups[-1]["params"]:
                if p.dtype not in TYPES:
                    raise TypeError("AdamW takes float32, bfloat16 or float16 parameters, not %s" % p.dtype)
                if not dense(p):
                    raise ValueError("AdamW needs dense parameters")
        except Exception:
            self.param_groups.pop()
            raise

    def _eight(self, p):
        return self.state_bits == 8 and p.numel() >= self.min_8bit_size

    def _new_state(self, p):
        if not self._eight(p):
            return {"step": 0, "exp_avg": torch.zeros_like(p, dtype=torch.float32), "exp_avg_sq": torch.zeros_like(p, dtype=torch.float32)}
        n = _blocks(p.numel())
        return {"step": 0, "exp_avg": torch.zeros_like(p, dtype=torch.int8), "exp_avg_sq": torch.zeros_like(p, dtype=torch.uint8),
                "exp_avg_scale": torch.zeros(n, device=p.device), "exp_avg_sq_scale": torch.zeros(n, device=p.device)}

    @torch.no_grad()
    def step(self, closure=None):
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            # (before a state is made, whose memory would be the graph's)
            raise RuntimeError("an AdamW step cannot be captured into a HIP graph: every replay would be the same step")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            buckets = {}
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise RuntimeError("AdamW takes no sparse gradients")
                st = self.state[p]
                if not st:
                    st.update(self._new_state(p))
                if not (g.is_contiguous() and p.is_contiguous()) and g.stride() != p.stride():
                    g = torch.empty_like(p).copy_(g)
                # one call for everything that shares a type, a device, a kind of state and a step number
                key = (p.dtype, p.get_device(), "exp_avg_scale" in st, st["step"])
                buckets.setdefault(key, []).append((p, g, st))
            for (_, _, eight, step), items in buckets.items():
                params, grads, states = zip(*items)
                more = {}
                if eight:
                    more = {"exp_avg_scales": [s["exp_avg_scale"] for s in states], "exp_avg_sq_scales": [s["exp_avg_sq_scale"] for s in states]}
                adamw_step(params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], step + 1, lr=group["lr"],
                           betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], **more)
                for s in states:
                    s["step"] = step + 1
        return loss

    def load_state_dict(self, state_dict):
        """Takes the state of an AdamW with either kind of state (PyTorch's own among them) and converts it to this one's.  The
        states of other optimizers, and of PyTorch's with amsgrad, maximize or a weight decay that goes through the
        gradient, are refused.  Nothing is changed where that fails."""
        # as the last of the hooks before loading, so that the state is what the user's own made of it, and is there when
        # those after loading run
        hook = self.register_load_state_dict_pre_hook(AdamW._taken)
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()

    def _taken(self, state_dict):
        saved, groups = state_dict["state"], state_dict["param_groups"]
        if any("exp_avg" not in st or "exp_avg_sq" not in st or set(st) - _STATE_KEYS for st in saved.values()) \
                or any(k not in g for g in groups for k in _CONSTANTS):
            raise ValueError("not the state of an AdamW optimizer")
        for g in groups:
            theirs = _TORCH_KEYS & set(g)
            if theirs and "amsgrad" not in g:
                raise ValueError("the state of another optimizer than AdamW")     # of the same family, such as RAdam
            if g.get("amsgrad") or g.get("maximize") or (not g.get("decoupled_weight_decay", True) and g["weight_decay"] != 0):
                raise ValueError("this AdamW has no amsgrad, no maximize and no weight decay through the gradient")
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the state of an optimizer with other parameter groups")
        ids = [i for g in groups for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        # PyTorch casts every state tensor that it finds by its number to its parameter's type, which codes and scales must not be;
        # what stands under the parameter itself it takes as it is
        new = {p: self._converted(p, saved[i]) for i, p in zip(ids, params) if i in saved}
        return {"state": new, "param_groups": [{k: v for k, v in g.items() if k not in _TORCH_KEYS} for g in groups]}

    def _converted(self, p, st):
        new = self._new_state(p)
        new["step"] = int(st["step"])
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            old, old_scale = st[name].detach(), st.get(name + "_scale")
            if old.shape != p.shape:
                raise ValueError("the state of a parameter of shape %s has shape %s" % (tuple(p.shape), tuple(old.shape)))
            scale = new.get(name + "_scale")
            if old_scale is not None and scale is not None and old.stride() == new[name].stride():
                if old.dtype != new[name].dtype or old_scale.dtype != torch.float32 or old_scale.shape != scale.shape:
                    raise ValueError("not the codes and scales of an 8-bit state")
                new[name].copy_(old)
                scale.copy_(old_scale)
                continue
            values = dequantize_state(old, old_scale) if old_scale is not None else old.float()
            if scale is None:
                new[name].copy_(values)
            else:
                laid_out = torch.empty_like(p, dtype=torch.float32).copy_(values)
                codes, scales = quantize_state(laid_out, signed)
                new[name].copy_(codes)
                scale.copy_(scales)
        return new
