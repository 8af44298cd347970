"""AdamW over many tensors at once on B200 (hand-written sm_100a CUDA), its states in fp32 or in 8 bits. Use the
optimizer AdamW(params, ...), or adamw_step(...) on lists of tensors.

One step, in place, for every tensor of the lists (t counts the steps):
  g' = g * min(1, max_norm / (|all g| + 1e-6)), or g where max_norm is 0
  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
  p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
The step count is one int64 on the device, as lr may be one fp32: a step captured into a CUDA graph counts on when
it is replayed.  With max_norm, a norm that is not finite leaves everything as it is, the count included.

Parameters in fp32, bf16 or f16, gradients in their type or fp32.  A 16-bit parameter may have an fp32 master: the
step is then taken on it, and the parameter is its rounding (without one, updates below half a unit of the
parameter's last place are lost).

States in 8 bits: m and sqrt(v) as float8_e4m3fn and, for each group of 256 elements, an exponent byte for either;
a value is code * 2^(exponent - 127).  The group's largest magnitude lies in [128, 256), so 13 binades below it keep
3 bits of mantissa.  A step moves sqrt(v) and often m by far less than half a code, so both are rounded up or down by a
hash of the element's place and t, right on average (the same bits every run): rounding="random", which AdamW takes.
With "nearest" m's codes are the nearest ones, as one step alone would have them; over a run of steps m then stops
wherever (1 - b1) |g' - m| is below half a code (0.71 of a constant gradient for b1 0.9), and an element whose gradients
have ended keeps moving.  10 bytes a bf16 parameter are read and written where fp32 states take 22.  A group with a
value that is not finite reads back as NaN.

Kernels: kernel-rsi_b200/csrc/adamw.cu; C ABI: include/krsi_b200.h.
"""
import sys
import warnings
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
from _compat import compiling  # noqa: E402
from _ext import direct, ops  # noqa: E402

GROUP = 256
_warned = False


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
               max_norm=0.0, masters=None, exponents=None, rounding=None):
    """One AdamW step on lists of tensors, in place; step: an int64 CUDA tensor, counted on.  exp_avgs and exp_avg_sqs
    are fp32, or float8_e4m3fn codes of m and sqrt(v) with exponents (new_state() makes either).  masters: fp32
    copies of the 16-bit parameters (None, or an entry without elements, where there is none).  Returns the norm of
    all gradients where max_norm > 0, else None.  No two tensors may overlap.

    rounding: of m's 8-bit codes, "random" (right on average: what a run of steps needs) or "nearest" (right for a single
    step; over a run m stops short of its mean).  Where it is not given it is "nearest", with a warning."""
    if rounding is None:
        if exponents and not _warned and not compiling():
            _warn_nearest(exp_avgs)
    elif rounding not in ("random", "nearest"):
        raise ValueError(f'adamw_step: rounding must be "random" or "nearest", got {rounding!r}')
    device_lr = isinstance(lr, torch.Tensor)
    args = (params, grads, exp_avgs, exp_avg_sqs, masters or [], exponents or [], step, lr if device_lr else None,
            0.0 if device_lr else lr, betas[0], betas[1], eps, weight_decay, max_norm, rounding == "random")
    norm = NotImplemented if direct is None or compiling() else direct.adamw_step(*args)
    if norm is NotImplemented:
        norm = ops.adamw_step(*args)
    return norm if max_norm > 0 else None


def _warn_nearest(exp_avgs):
    global _warned
    if any(m.dtype == torch.float8_e4m3fn for m in exp_avgs):
        _warned = True
        warnings.warn('adamw_step: 8-bit states are rounded to nearest, which is right for a single step only; a run of '
                      'steps needs rounding="random" ("nearest" is this, without the warning)', stacklevel=3)


def new_state(p, bits=32):
    """Zero states of a parameter: (exp_avg, exp_avg_sq, exponents), exponents without elements for 32 bits."""
    groups = -(-p.numel() // GROUP) if bits == 8 else 0
    exponents = torch.zeros(groups, 2, dtype=torch.uint8, device=p.device)
    dtype = torch.float8_e4m3fn if bits == 8 else torch.float32
    exp_avg, exp_avg_sq = (torch.zeros(p.shape, dtype=dtype, device=p.device) for _ in range(2))
    return exp_avg, exp_avg_sq, exponents


def dequantise(exp_avg, exp_avg_sq, exponents):
    """(m, v) in fp32 that 8-bit states stand for (torch ops)."""
    scale = torch.where(exponents == 255, float("nan"), torch.exp2(exponents.double() - 127))
    scale = scale.repeat_interleave(GROUP, 0)[:exp_avg.numel()]
    m, r = ((q.reshape(-1).double() * scale[:, k]).view(q.shape) for k, q in enumerate((exp_avg, exp_avg_sq)))
    return m.float(), r.square().float()


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's role on adamw_step(): each parameter group is one call.

    bits: of the states (8: m and sqrt(v) rounded at random, right on average over a run for b1 up to 0.999); parameters
    with fewer than min_8bit_size elements keep fp32 ones.  master: keep an fp32 master of each 16-bit parameter.  max_norm: clip by the norm of the group's gradients (0: not), which is the model's
    where there is one group alone (else torch.nn.utils.clip_grad_norm_ before the step); grad_norm holds the last
    step's, one a group.  lr may be a 0-dim fp32 CUDA tensor.  Parameters without a gradient are left
    alone; the step counts the group's calls, not each parameter's.  States are made by the first step, or by
    init_states(), which has to come before a step is captured into a CUDA graph."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_norm=0.0, bits=32,
                 master=False, min_8bit_size=4096):
        if bits not in (8, 32):
            raise ValueError(f"AdamW: bits must be 8 or 32, got {bits}")
        if not isinstance(lr, torch.Tensor) and lr < 0:
            raise ValueError(f"AdamW: lr must not be negative, got {lr}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {betas}")
        if eps < 0 or max_norm < 0 or weight_decay < 0:
            raise ValueError("AdamW: eps, max_norm and weight_decay must not be negative")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_norm=max_norm,
                                      bits=bits, master=master, min_8bit_size=min_8bit_size))
        self.grad_norm = []

    def init_states(self):
        """Makes the states that are missing."""
        for group in self.param_groups:
            for p in group["params"]:
                self._state(group, p)
        return self

    def _step_of(self, group, device):
        step = group.get("step")
        if step is None or step.device != device:
            self._no_capture()
            group["step"] = step = torch.zeros((), dtype=torch.int64, device=device) if step is None else step.to(device)
        return step

    @staticmethod
    def _no_capture():
        if torch.cuda.is_current_stream_capturing():   # a replay would make them anew
            raise RuntimeError("AdamW: call init_states(), or step() once, before capturing a step")

    @torch.no_grad()
    def _state(self, group, p):
        self._step_of(group, p.device)
        state = self.state[p]
        if "exp_avg" not in state:
            self._no_capture()
            bits = 8 if group["bits"] == 8 and p.numel() >= group["min_8bit_size"] else 32
            state["exp_avg"], state["exp_avg_sq"], state["exponents"] = new_state(p, bits)
            master = group["master"] and p.dtype != torch.float32
            state["master"] = p.detach().float().contiguous() if master else torch.zeros(0, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.grad_norm = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                self.grad_norm.append(None)
                continue
            states = [self._state(group, p) for p in params]
            columns = {k: [s[k] for s in states] for k in ("exp_avg", "exp_avg_sq", "master", "exponents")}
            self.grad_norm.append(adamw_step(
                params, [p.grad for p in params], columns["exp_avg"], columns["exp_avg_sq"], group["step"],
                lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                max_norm=group["max_norm"], masters=columns["master"], exponents=columns["exponents"],
                rounding="random"))
        return loss

    def load_state_dict(self, state_dict):
        """The base class casts states to their parameter's type; they keep their own here.  It leaves a group's tensors
        where the dictionary has them; the step count and a tensor lr go to the group's parameters' device."""
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            for key in ("step", "lr"):
                if isinstance(group.get(key), torch.Tensor) and group["params"]:
                    group[key] = group[key].to(group["params"][0].device)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for key, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, torch.Tensor):
                    self.state[p][key] = value.to(p.device, copy=True)


def reference(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
              max_norm=0.0):
    """The step in torch ops on lists of tensors with fp32 states: the new (params, exp_avgs, exp_avg_sqs) in fp32."""
    t, clip = int(step) + 1, 1.0
    if max_norm > 0:
        norm = torch.stack([g.float().norm() for g in grads]).norm()
        clip = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    out = []
    for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs):
        g = g.float() * clip
        m = betas[0] * m + (1 - betas[0]) * g
        v = betas[1] * v + (1 - betas[1]) * g * g
        root = v.sqrt() / (1 - betas[1] ** t) ** 0.5 + eps
        out.append((p.float() * (1 - lr * weight_decay) - lr / (1 - betas[0] ** t) * m / root, m, v))
    return tuple(map(list, zip(*out)))


def selftest():
    """adamw_step against reference() on three tensors; the largest difference of the parameters."""
    params = [torch.randn(s, device="cuda") for s in ((1152, 512), (77,), (3, 5))]
    grads = [torch.randn_like(p) for p in params]
    states = [new_state(p) for p in params]
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    want, _, _ = reference(params, grads, [s[0] for s in states], [s[1] for s in states], step, lr=1e-3)
    adamw_step(params, grads, [s[0] for s in states], [s[1] for s in states], step, lr=1e-3)
    err = max((a - b).abs().max().item() for a, b in zip(params, want))
    return {"ok": err < 1e-6, "max": err}


if __name__ == "__main__":
    print(selftest())
