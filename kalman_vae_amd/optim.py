"""AdamW (decoupled weight decay) on a hand-written HIP kernel (csrc/adamw.hip): all tensors of a
model in one launch per 48 of them, with states in float32 or in 8 bits.

The reference trains with torch.optim.Adam (examples/train.py:67, 126-131); ``AdamW`` here is used the same way, also
in ``parallel.DataParallelStep``.
"""
import torch

from . import _capi as capi

BLOCK = 256              # elements of an 8-bit state that share a scale


def state_blocks(numel):
    """Scales of an 8-bit state of `numel` elements."""
    return -(-numel // BLOCK)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2, masters=None, seed=0):
    """One AdamW update of a list of tensors, in place:

        m = b1 m + (1-b1) g,  v = b2 v + (1-b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    ``params`` and ``grads``: contiguous GPU tensors of one type (float32, bfloat16 or float16) on one
    device; none of the tensors that are written may share memory.  ``exp_avgs`` and ``exp_avg_sqs``: float32 tensors holding m and v, or pairs
    ``(codes, scales)`` holding m and sqrt(v) in 8 bits: codes of torch.float8_e4m3fn with the
    parameter's number of elements and one float32 scale per 256 of them (``state_blocks``).  8-bit
    states are rounded stochastically by a hash of ``seed``, ``step`` and the element's place in the
    list: the same call gives the same bits.  A gradient that is not finite spoils the states of its
    element (32 bits) or of its 256 (8 bits), so such an update has to be left out.  ``masters``: float32 copies of 16-bit parameters that take the update, of which the
    parameter is the rounded value; without them the update is rounded to the parameter's type.

    ``step``: the number of this update, from 1; or an int64 tensor of one element on the device that
    holds it (then the call can be captured into a graph and replayed), in which case ``lr`` may be a
    float32 tensor of one element too.  Arithmetic is float32; nothing is allocated."""
    capi.torch_entry().adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, *betas, eps, weight_decay,
                                  masters, int(seed) & 0xFFFFFFFF, False)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s update through ``adamw_step``: ``state_bits=32`` (float32 states) or 8
    (2 bytes per element instead of 8).

    16-bit parameters keep a float32 copy in the state that takes the updates; an element of the
    parameter that was changed from outside (weights loaded, clipped or set between steps, by
    whatever means) is taken over into it.  Gradients have the parameter's type; parameters are
    float32, bfloat16 or float16, contiguous and on a GPU.
    ``capturable=True`` keeps the step count of each group on the device, so that ``step()`` can be
    captured into a HIP graph and replayed (the first step, which makes the states, outside the
    capture; a loaded state dict needs a new one); ``lr`` may then be a float32 tensor that the caller
    changes between replays, and every parameter of the group must have a gradient from the first
    step on, or never."""

    _former_counts = ()

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
        parameter's type: the states are taken over in their own.  A step count and a rate that are
        tensors go to the parameters' device, from wherever they were loaded."""
        super().load_state_dict(state_dict)
        params = [p for g in self.param_groups for p in g["params"]]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for p, i in zip(params, ids):
            for name, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, torch.Tensor):
                    self.state[p][name] = value.detach().to(p.device, copy=True)
        for g, saved in zip(self.param_groups, state_dict["param_groups"]):
            for name in ("step", "lr"):
                if isinstance(saved.get(name), torch.Tensor):
                    g[name] = saved[name].detach().to(g["params"][0].device, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check_capture()
        salt = 0                        # lists of one step draw different random bits
        for group in self.param_groups:
            lists = {}
            if not group["capturable"] and group.get("step") is not None:
                # no longer capturable: the device's count is the one that replays have advanced (it is kept, as
                # graphs that were captured write it)
                self._former_counts += (group["step"],)
                count, group["step"] = int(group["step"]), None
                for p in group["params"]:
                    if self.state.get(p):
                        self.state[p]["step"] = count
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                lists.setdefault((p.device, p.dtype, state["step"] + 1), []).append((p, state))
            if group["capturable"] and lists:
                self._device_step(group, lists)
            for n, ((device, dtype, step), entries) in enumerate(lists.items()):
                pair = lambda name: ([(s[name], s[name + "_scale"]) for _, s in entries]  # noqa: E731
                                     if group["state_bits"] == 8 else [s[name] for _, s in entries])
                try:
                    capi.torch_entry().adamw_step(
                        [p for p, _ in entries],
                        [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p, _ in entries],
                        pair("exp_avg"), pair("exp_avg_sq"), group["step"] if group["capturable"] else step,
                        group["lr"], *group["betas"], group["eps"], group["weight_decay"],
                        [s["master"] for _, s in entries] if dtype != torch.float32 else None,
                        (int(group["seed"]) + 0x51ED2701 * salt) & 0xFFFFFFFF, True)
                except Exception:                    # refused: no step has been made
                    if group["capturable"] and n == 0:
                        group["step"].sub_(1)
                    raise
                for _, state in entries:
                    state["step"] = step
                salt += 1
        return loss

    def _check_capture(self):
        """A replay repeats what was captured: a count that the host passes would stand still, states that
        are made inside the capture would be cleared each time."""
        if not (torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()):
            return
        for group in self.param_groups:
            given = [p for p in group["params"] if p.grad is not None]
            if given and not group["capturable"]:
                raise RuntimeError("AdamW.step() is being captured into a graph: this needs capturable=True")
            if not all(self.state.get(p) for p in given):
                raise RuntimeError("AdamW.step() is being captured into a graph, but a parameter has no state yet: "
                                   "run a step before the capture")

    def _device_step(self, group, lists):
        """Advance the group's step count on the device (one launch, captured with the step)."""
        if len({step for _, _, step in lists}) > 1 or len({device for device, _, _ in lists}) > 1:
            raise RuntimeError("capturable=True: the parameters of a group share one step count on one "
                               "device, so each needs a gradient in every step, or in none")
        if group.get("step") is None:
            device, _, step = next(iter(lists))
            group["step"] = torch.full((1,), step - 1, dtype=torch.int64, device=device)
        group["step"].add_(1)
