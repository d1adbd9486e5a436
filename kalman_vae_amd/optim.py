"""AdamW (decoupled weight decay) on a hand-written HIP kernel (csrc/adamw.hip): all tensors of a
model in one launch per 48 of them, with states in float32 or in 8 bits.

The reference trains with torch.optim.Adam (examples/train.py:67, 126-131); ``AdamW`` here is used the same way, also
in ``parallel.DataParallelStep``.
"""
import ctypes as C

import torch

from . import _capi as capi
from .sequence_ops import _on, _stream

BLOCK = 256              # elements of an 8-bit state that share a scale
MAX_TENSORS = 48         # tensors of one launch


def state_blocks(numel):
    """Scales of an 8-bit state of `numel` elements."""
    return -(-numel // BLOCK)


def _check_list(name, tensors, like, dtypes, device):
    """Addresses of `tensors`: as many as `like`, of the same sizes, contiguous, on `device`."""
    if len(tensors) != len(like):
        raise ValueError(f"{len(tensors)} {name} for {len(like)} parameters")
    for t, p in zip(tensors, like):
        if t.dtype not in dtypes:
            raise TypeError(f"{name}: expected {' or '.join(map(str, dtypes))}, got {t.dtype}")
        if t.numel() != p.numel():
            raise ValueError(f"{name}: {t.numel()} elements for a parameter of {p.numel()}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.device != device:
            capi.require_gpu(t)
            raise ValueError(f"{name} on {t.device}, parameters on {device}")
    return [t.data_ptr() for t in tensors]


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2, masters=None, seed=0):
    """One AdamW update of a list of tensors, in place:

        m = b1 m + (1-b1) g,  v = b2 v + (1-b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    ``params`` and ``grads``: contiguous GPU tensors of one type (float32, bfloat16 or float16) on one
    device.  ``exp_avgs`` and ``exp_avg_sqs``: float32 tensors holding m and v, or pairs
    ``(codes, scales)`` holding m and sqrt(v) in 8 bits: codes of torch.float8_e4m3fn with the
    parameter's number of elements and one float32 scale per 256 of them (``state_blocks``).  8-bit
    states are rounded stochastically by a hash of ``seed``, ``step`` and the element's place in the
    list: the same call gives the same bits.  ``masters``: float32 copies of 16-bit parameters that take the update, of which the
    parameter is the rounded value; without them the update is rounded to the parameter's type.

    ``step``: the number of this update, from 1; or an int64 tensor of one element on the device that
    holds it (then the call can be captured into a graph and replayed), in which case ``lr`` may be a
    float32 tensor of one element too.  Arithmetic is float32; nothing is allocated."""
    if not params:
        return
    device, dtype = params[0].device, params[0].dtype
    capi.require_gpu(params[0])
    code = capi.sequence_dtype_code(dtype)
    p_at = _check_list("parameters", params, params, (dtype,), device)
    if len(set(p_at)) != len(p_at):
        # (empty tensors have no address of their own and take no part)
        full = [a for a, p in zip(p_at, params) if p.numel()]
        if len(set(full)) != len(full):
            raise ValueError("a parameter appears twice in the list")
    g_at = _check_list("gradients", grads, params, (dtype,), device)
    bits = 8 if exp_avgs and isinstance(exp_avgs[0], (tuple, list)) else 32
    if any(isinstance(e, (tuple, list)) != (bits == 8) for e in (*exp_avgs, *exp_avg_sqs)):
        raise TypeError("states are all float32 tensors or all (codes, scales) pairs")
    if bits == 8:
        code_types, f32 = (torch.float8_e4m3fn,), (torch.float32,)
        columns = []
        for name, pairs in (("exp_avgs", exp_avgs), ("exp_avg_sqs", exp_avg_sqs)):
            columns.append(_check_list(name, [c for c, _ in pairs], params, code_types, device))
            scales = [s for _, s in pairs]
            for s, p in zip(scales, params):
                if s.dtype != torch.float32 or s.numel() != state_blocks(p.numel()):
                    raise ValueError(f"{name}: {state_blocks(p.numel())} float32 scales for a parameter of "
                                     f"{p.numel()}, got {s.numel()} of {s.dtype}")
                if not s.is_contiguous() or s.device != device:
                    raise ValueError(f"{name}: scales must be contiguous and on {device}")
            columns.append([s.data_ptr() for s in scales])
        m_at, ms_at, v_at, vs_at = columns
    else:
        m_at = _check_list("exp_avgs", exp_avgs, params, (torch.float32,), device)
        v_at = _check_list("exp_avg_sqs", exp_avg_sqs, params, (torch.float32,), device)
        ms_at = vs_at = [0] * len(params)
    if masters is not None:
        if dtype == torch.float32:
            raise ValueError("masters belong to 16-bit parameters")
        w_at = _check_list("masters", masters, params, (torch.float32,), device)
    else:
        w_at = [0] * len(params)
    d = capi.AdamW(dtype=code, state_bits=bits, seed=int(seed) & 0xFFFFFFFF, beta1=betas[0], beta2=betas[1],
                   eps=eps, weight_decay=weight_decay)
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != device:
            raise ValueError("step must be an int64 tensor of one element on the parameters' device")
        d.step_device = step.data_ptr()
    elif step < 1:
        raise ValueError(f"step counts from 1, got {step}")
    else:
        d.step = step
    if isinstance(lr, torch.Tensor):
        if not isinstance(step, torch.Tensor) or lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != device:
            raise ValueError("lr as a tensor: float32, one element, on the parameters' device, with step a tensor too")
        d.lr_device = lr.data_ptr()
    else:
        d.lr = lr
    rows = [row for row in zip([p.numel() for p in params], p_at, g_at, m_at, v_at, ms_at, vs_at, w_at) if row[0]]
    lib = capi.load()
    with _on(device):
        stream, first_block = _stream(device), 0
        for i in range(0, len(rows), MAX_TENSORS):
            part = rows[i:i + MAX_TENSORS]
            table = (C.c_int64 * (8 * len(part)))(*[v for row in part for v in row])
            d.tensors, d.count, d.first_block = C.addressof(table), len(part), first_block
            capi.check(lib.kvae_adamw_step(C.byref(d), stream))
            first_block += sum(-(-row[0] // BLOCK) for row in part)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s update through ``adamw_step``: ``state_bits=32`` (float32 states) or 8
    (2 bytes per element instead of 8).

    16-bit parameters keep a float32 copy in the state that takes the updates.  Gradients have the
    parameter's type; parameters are float32, bfloat16 or float16, contiguous and on a GPU.
    ``capturable=True`` keeps the step count of each group on the device, so that ``step()`` can be
    captured into a HIP graph and replayed; ``lr`` may then be a float32 tensor that the caller
    changes between replays, and every parameter of the group must have a gradient from the first
    step on, or never."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 seed=0, capturable=False):
        if not isinstance(lr, torch.Tensor) and lr < 0:
            raise ValueError(f"invalid lr: {lr}")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("lr as a tensor needs capturable=True")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"invalid betas: {betas}")
        if eps < 0 or weight_decay < 0:
            raise ValueError(f"invalid eps or weight_decay: {eps}, {weight_decay}")
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits is 32 or 8, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, seed=seed, capturable=capturable))

    def _new_state(self, p, group):
        if not p.is_contiguous():
            raise ValueError("AdamW needs contiguous parameters")
        capi.require_gpu(p)
        capi.sequence_dtype_code(p.dtype)
        state = {"step": 0}
        if group["state_bits"] == 8:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device)
                state[name + "_scale"] = torch.full((state_blocks(p.numel()),), 2.0 ** -126,
                                                    dtype=torch.float32, device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if p.dtype != torch.float32:
            state["master"] = p.detach().float()
        return state

    def load_state_dict(self, state_dict):
        """As torch.optim.Optimizer, which would convert every floating-point state to the
        parameter's type: the states are taken over in their own."""
        super().load_state_dict(state_dict)
        params = [p for g in self.param_groups for p in g["params"]]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for p, i in zip(params, ids):
            for name, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, torch.Tensor):
                    self.state[p][name] = value.detach().to(p.device, copy=True)
        for g, saved in zip(self.param_groups, state_dict["param_groups"]):
            if isinstance(saved.get("step"), torch.Tensor):
                g["step"] = saved["step"].detach().to(g["params"][0].device, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        salt = 0                        # lists of one step draw different random bits
        for group in self.param_groups:
            lists = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                state["step"] += 1
                lists.setdefault((p.device, p.dtype, state["step"]), []).append((p, state))
            if group["capturable"]:
                self._device_step(group, lists)
            for (device, dtype, step), entries in lists.items():
                pair = lambda name: ([(s[name], s[name + "_scale"]) for _, s in entries]  # noqa: E731
                                     if group["state_bits"] == 8 else [s[name] for _, s in entries])
                adamw_step([p for p, _ in entries],
                           [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p, _ in entries],
                           pair("exp_avg"), pair("exp_avg_sq"),
                           group["step"] if group["capturable"] else step, lr=group["lr"],
                           betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                           masters=[s["master"] for _, s in entries] if dtype != torch.float32 else None,
                           seed=group["seed"] + 0x51ED2701 * salt)
                salt += 1
        return loss

    def _device_step(self, group, lists):
        """Advance the group's step count on the device (one launch, captured with the step)."""
        if len({step for _, _, step in lists}) > 1 or len({device for device, _, _ in lists}) > 1:
            raise RuntimeError("capturable=True: the parameters of a group share one step count on one "
                               "device, so each needs a gradient in every step, or in none")
        if not lists:
            return
        if group.get("step") is None:
            device = next(iter(lists))[0]
            group["step"] = torch.zeros(1, dtype=torch.int64, device=device)
        group["step"].add_(1)
