"""Dynamics-parameter ("weight") networks: (t,B,a_dim) -> softmax (t,B,K): the reference's
LSTM and perceptron, and a stack of gated linear recurrences.

Ordinary PyTorch modules whose hot parts run on the package's HIP kernels when
the tensors are float32 on a GPU (LSTM recurrence for whole-sequence calls, the
Linear+softmax head); on the CPU they are plain torch.  Parameter names match the
reference (kvae/dynamics_parameter_network.py:18-90) so its checkpoints load:
``lstm.*`` + ``linear.*`` for the LSTM model, ``layers.<i>.*`` for the MLP.
"""
import contextlib

import torch
import torch.nn as nn

from . import _capi as capi
from . import lstm_function
from .sequence_ops import (gated_scan, gated_scan_step, linear_8bit, quantize_rows, rms_norm,
                           rms_norm_quantized)


class LSTMModel(nn.Module):
    """nn.LSTM -> Linear -> softmax with the recurrent state cached on the
    module between calls, so that feeding the sequence one step at a time
    equals feeding it whole."""

    def __init__(self, input_dim, output_dim, hidden_dim, num_layers):
        super().__init__()
        self.hidden_dim = hidden_dim
        self.num_layers = num_layers
        self.lstm = nn.LSTM(input_dim, hidden_dim, num_layers=num_layers)
        self.linear = nn.Linear(hidden_dim, output_dim)
        self._hidden = None
        self.count = 0
        # whole-sequence calls on a GPU run the recurrence on the package's HIP
        # kernels (float32, hidden_dim a multiple of 32); step-by-step calls and
        # everything else use torch.nn.LSTM
        self.use_hip_recurrence = True

    @property
    def hidden(self):
        """(h_n, c_n) carried between calls, each (num_layers, B, hidden_dim), or None."""
        if isinstance(self._hidden, lstm_function.LastState):
            self._hidden = self._hidden.get()
        return self._hidden

    @hidden.setter
    def hidden(self, value):
        self._hidden = value

    def clear_hidden_state(self):
        self.hidden = None
        self.count = 0

    def reset_hidden_state(self, batch_size, device, dtype):
        shape = (self.num_layers, batch_size, self.hidden_dim)
        self.hidden = (torch.zeros(shape, dtype=dtype, device=device),
                       torch.zeros(shape, dtype=dtype, device=device))
        self.count = 0

    def forward(self, x, lead=False):
        """x (t,B,a_dim) -> weights (t,B,K); lead=True prepends the uniform weights
        of the step before the first observation: (t+1,B,K)."""
        self.count += 1
        if (self.use_hip_recurrence and self.hidden is None and x.size(0) > 1
                and lstm_function.supported(x, self.hidden_dim)):
            # whole sequence from a fresh state: recurrence on the HIP kernels (the default
            # network as one node: its backward forms the head's adjoint inside the upper
            # layer's kernel)
            fused = lstm_function.fused_lstm_head(x, self.lstm, self.linear, lead)
            if fused is not None:
                self.hidden = fused[1]
                return fused[0]
            h, hidden = lstm_function.fused_lstm(x, self.lstm)
            self.hidden = (hidden if isinstance(hidden, lstm_function.LastState)
                           else (hidden[0].detach(), hidden[1].detach()))
            return lstm_function.softmax_head(h, self.linear, lead)
        if (self.use_hip_recurrence and not torch.is_grad_enabled()
                and lstm_function.persistent_supported(x, self.lstm)):
            # inference from the carried state (the step-by-step masked filter): the
            # persistent kernel continues from self.hidden, no library RNN call
            h, self.hidden = lstm_function.lstm2_nograd(x, self.lstm, self.hidden)
            return lstm_function.softmax_head(h, self.linear, lead)
        if self.hidden is None:
            self.reset_hidden_state(x.size(1), device=x.device, dtype=x.dtype)
        h, self.hidden = self._library_lstm(x)
        return lstm_function.softmax_head(h, self.linear, lead)

    def _library_lstm(self, x):
        """self.lstm(x, self.hidden) through torch.  MIOpen refuses the backward of an LSTM
        that ran in eval mode, so a run in eval mode that records a gradient (masked
        sequences of an evaluation that differentiates) takes PyTorch's native kernels."""
        if x.is_cuda and not self.training and torch.is_grad_enabled():
            with torch.backends.cudnn.flags(enabled=False):
                return self.lstm(x, self.hidden)
        return self.lstm(x, self.hidden)

    def inference_stepper(self, x):
        """For a caller that feeds one step at a time without a gradient (the masked
        filter): an object whose ``step(x_t (B,a_dim), out (B,K))`` equals
        ``out.copy_(self(x_t[None])[0])`` with fewer launches and no per-step tensors, or
        None when that form does not apply.  Call ``finish_steps`` afterwards so that the
        module carries the state on, as after the equivalent forward calls."""
        if not self.use_hip_recurrence:
            return None
        return lstm_function.LSTM2HeadStepper.make(x, self.lstm, self.linear, self.hidden)

    def finish_steps(self, stepper, steps):
        self.hidden = stepper.hidden
        self.count += steps

    is_recurrent = True


class MLPModel(nn.Module):
    """num_layers Linear layers with ReLU between them, softmax on top."""

    def __init__(self, input_dim, output_dim, hidden_dim, num_layers):
        super().__init__()
        self.hidden_dim = hidden_dim
        self.num_layers = num_layers
        self.input_dim = input_dim
        self.output_dim = output_dim
        # The first layer always maps to hidden_dim, also when it is the only
        # layer (dynamics_parameter_network.py:70-76 tests i == 0 first).
        self.layers = nn.ModuleList()
        for i in range(num_layers):
            fan_in = input_dim if i == 0 else hidden_dim
            fan_out = output_dim if (i == num_layers - 1 and i != 0) else hidden_dim
            self.layers.append(nn.Linear(fan_in, fan_out))

    def clear_hidden_state(self):
        pass

    def reset_hidden_state(self, batch_size, device, dtype):
        pass

    def forward(self, x, lead=False):
        last = len(self.layers) - 1
        for i, layer in enumerate(self.layers):
            if i == last:
                return lstm_function.softmax_head(x, layer, lead)
            x = torch.relu(lstm_function.linear(x, layer))

    is_recurrent = False


def _device_of(x):
    """x's device as the current one, for what launches on the current device's stream."""
    if not x.is_cuda or x.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(x.device)


def _plain_norm(x, weight, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight


def _plain_scan(u, state):
    """gated_scan by its definition, one step after the other (CPU and float64)."""
    x, forget, gate = u.chunk(3, dim=-1)
    f, keep = torch.sigmoid(forget), torch.sigmoid(-forget)
    c = torch.zeros_like(x[0]) if state is None else state
    steps = []
    for t in range(u.shape[0]):
        c = f[t] * c + keep[t] * x[t]
        steps.append(c)
    return torch.stack(steps) * torch.nn.functional.silu(gate), c


class GatedBlock(nn.Module):
    """norm -> projection to [x | forget | gate] -> gated recurrence -> projection back."""

    def __init__(self, hidden_dim):
        super().__init__()
        self.norm = nn.Parameter(torch.ones(hidden_dim))
        self.proj = nn.Linear(hidden_dim, 3 * hidden_dim)
        self.out = nn.Linear(hidden_dim, hidden_dim)
        with torch.no_grad():                  # gates that mostly remember to begin with
            self.proj.bias[hidden_dim:2 * hidden_dim] += 1.0


class GatedModel(nn.Module):
    """A stack of gated linear recurrences with pre-norm residuals:

        h = embed(x);  per block: h += out(scan(proj(norm(h))));  weights = softmax(linear(norm(h)))

    The recurrent alternative to ``LSTMModel`` whose time axis holds no matrix product: all
    projections run over the whole sequence at once and the recurrence between them is a scan
    (``gated_scan``), which also runs parallel in time.  Used like the LSTM: the state is cached on
    the module between calls, and feeding a sequence one step at a time equals feeding it whole.
    On a GPU in float32, bfloat16 or float16 the norms and scans are the package's HIP kernels; on the
    CPU and in float64 the module is plain torch.

    After ``eight_bit()`` calls that record no gradient run the blocks' projections as ``linear_8bit``
    on the norm's 8-bit output.  The reference has no
    counterpart of this network (kvae/dynamics_parameter_network.py:18-90 has the LSTM and the MLP)."""

    eps = 1e-6
    is_recurrent = True

    def __init__(self, input_dim, output_dim, hidden_dim, num_layers):
        super().__init__()
        if num_layers < 1:
            raise ValueError(f"num_layers must be at least 1, got {num_layers}")
        self.hidden_dim = hidden_dim
        self.num_layers = num_layers
        self.embed = nn.Linear(input_dim, hidden_dim)
        self.blocks = nn.ModuleList(GatedBlock(hidden_dim) for _ in range(num_layers))
        self.norm = nn.Parameter(torch.ones(hidden_dim))
        self.linear = nn.Linear(hidden_dim, output_dim)
        self.use_hip_kernels = True
        self._states = None                    # one (B,H) per block, or None
        self._eight = None                     # see eight_bit()
        self.count = 0

    # -- state carried between calls --------------------------------------------------------
    @property
    def hidden(self):
        """The state carried between calls, (num_layers, B, hidden_dim), or None."""
        return None if self._states is None else torch.stack(self._states)

    @hidden.setter
    def hidden(self, value):
        self._states = None if value is None else list(value.unbind(0))

    def clear_hidden_state(self):
        self._states = None
        self.count = 0

    def reset_hidden_state(self, batch_size, device, dtype):
        self.hidden = torch.zeros(self.num_layers, batch_size, self.hidden_dim, device=device,
                                  dtype=torch.float32 if dtype in capi.SEQUENCE_DTYPES else dtype)
        self.count = 0

    # -- 8-bit serving form -----------------------------------------------------------------
    def eight_bit(self, on=True):
        """Turn the 8-bit form of the blocks' projections on (or off) for the parameters as they are.
        Calls without a gradient then make the codes, and one float32 scale per output, from the
        weights that the model has when they run, so that none answers from former ones however they
        were changed; an ``inference_stepper`` makes them once for its steps.  A change that autograd
        records (in place, replaced or loaded parameters) ends the form: such calls raise until this
        is called again.  Moving or converting the module turns it off.  Returns self."""
        self._eight = None
        if on:
            capi.require_gpu(self.norm)
            capi.sequence_dtype_code(self.norm.dtype)
            if self.hidden_dim > capi.NORM_MAX_WIDTH:
                raise NotImplementedError(f"up to {capi.NORM_MAX_WIDTH} channels, got {self.hidden_dim}")
            self._eight = [[[(name, p, p._version) for name, p in layer._parameters.items()]
                            for layer in (block.proj, block.out)] for block in self.blocks]
        return self

    def _apply(self, fn, recurse=True):
        self._eight = None                     # moved or converted parameters
        return super()._apply(fn, recurse)

    def _check_unchanged(self, known):
        """Raise where autograd's records show a change since eight_bit() noted `known`."""
        for block, layers in zip(self.blocks, known):
            for layer, params in zip((block.proj, block.out), layers):
                if any(layer._parameters.get(name) is not p or p._version != version for name, p, version in params):
                    raise RuntimeError("the parameters have changed since eight_bit(): call it again")

    def _codes_8bit(self):
        """[(weight codes, scales, bias) of proj and out] of every block, from the present parameters."""
        self._check_unchanged(self._eight)
        return [[(*quantize_rows(layer.weight), layer.bias.float()) for layer in (block.proj, block.out)]
                for block in self.blocks]

    # -- forward ----------------------------------------------------------------------------
    def _on_kernels(self, x):
        return (self.use_hip_kernels and x.is_cuda and x.dtype in capi.SEQUENCE_DTYPES
                and self.hidden_dim <= capi.NORM_MAX_WIDTH)

    def _use_8bit(self, x):
        return self._eight is not None and self._on_kernels(x) and not torch.is_grad_enabled()

    def _stack(self, x, scan, codes):
        """The last norm's output; scan(i, u) runs block i's recurrence.  codes: see _codes_8bit; None
        for the full form."""
        kernels = self._on_kernels(x)
        h, branch = lstm_function.linear(x, self.embed), None
        for i, block in enumerate(self.blocks):
            if codes is not None:
                (w_in, s_in, b_in), (w_out, s_out, b_out) = codes[i]
                if branch is None:
                    q, scale = rms_norm_quantized(h, block.norm, eps=self.eps)
                else:
                    q, scale, h = rms_norm_quantized(branch, block.norm, residual=h, eps=self.eps)
                # (bfloat16 between the products: its rounding is far below that of 8 bits)
                y = scan(i, linear_8bit(q, scale, w_in, s_in, bias=b_in, dtype=torch.bfloat16))
                branch = linear_8bit(*quantize_rows(y), w_out, s_out, bias=b_out, dtype=x.dtype)
            else:
                n, h = self._norm(h, branch, block.norm, kernels)
                branch = lstm_function.linear(scan(i, lstm_function.linear(n, block.proj)), block.out)
        return self._norm(h, branch, self.norm, kernels)[0]

    def _norm(self, h, branch, weight, kernels):
        """(norm of h + branch, h + branch)"""
        if not kernels:
            h = h if branch is None else h + branch
            return _plain_norm(h, weight, self.eps), h
        if branch is None:
            return rms_norm(h, weight, eps=self.eps), h
        return rms_norm(branch, weight, residual=h, eps=self.eps)

    def forward(self, x, lead=False):
        """x (t,B,a_dim) -> weights (t,B,K); lead=True prepends the uniform weights
        of the step before the first observation: (t+1,B,K)."""
        self.count += 1
        kernels = self._on_kernels(x)
        states, ends = self._states, []
        fresh = states is None and x.size(0) > 1

        def scan(i, u):
            first = None if states is None else states[i]
            y, end = gated_scan(u, first) if kernels else _plain_scan(u, first)
            # (as in LSTMModel: a whole sequence from a fresh state leaves a state without a graph)
            ends.append(end.detach() if fresh else end)
            return y

        with _device_of(x):
            n = self._stack(x, scan, self._codes_8bit() if self._use_8bit(x) else None)
            self._states = ends
            return lstm_function.softmax_head(n, self.linear, lead)

    def inference_stepper(self, x):
        """For a caller that feeds one step at a time without a gradient (the masked filter): an
        object whose ``step(x_t (B,a_dim), out (B,K))`` equals ``out.copy_(self(x_t[None])[0])`` with
        the state updated in place (``gated_scan_step``), or None when that form does not apply.
        The parameters must not change before its last step (in the 8-bit form it holds their codes).
        Call ``finish_steps`` afterwards so that the module carries the state on."""
        if (torch.is_grad_enabled() or x.dim() != 2 or x.dtype != torch.float32 or not self._on_kernels(x)
                or not lstm_function.head_supported(x.new_empty(1, self.hidden_dim), self.linear)):
            return None
        return GatedStepper(self, x)

    def finish_steps(self, stepper, steps):
        self._states = stepper.states
        self.count += steps


class GatedStepper:
    """See ``GatedModel.inference_stepper``."""

    def __init__(self, model, x):
        self.model, B = model, x.shape[0]
        self.states = [torch.zeros(B, model.hidden_dim, device=x.device) if model._states is None
                       else model._states[i].clone() for i in range(model.num_layers)]
        self.known, self.codes = None, None
        if model._use_8bit(x):
            self.known, self.codes = model._eight, model._codes_8bit()

    @torch.no_grad()
    def step(self, x, out):
        """x (B,P) -> out (B,K), contiguous float32; advances the carried state."""
        model = self.model
        if not (out.is_contiguous() and out.shape == (x.shape[0], model.linear.out_features)
                and x.dtype == out.dtype == torch.float32):
            raise ValueError("GatedStepper.step: x (B,P) and contiguous out (B,K) must be float32")
        if self.known is not None:
            model._check_unchanged(self.known)
        with _device_of(x):
            n = model._stack(x, lambda i, u: gated_scan_step(u, self.states[i]), self.codes)
            W, b = model.linear.weight.contiguous(), model.linear.bias.contiguous()
            capi.check(capi.load().kvae_softmax_head_forward(
                n.shape[0], model.hidden_dim, W.shape[0], n.data_ptr(), W.data_ptr(), b.data_ptr(),
                out.data_ptr(), 0, capi.current_stream_ptr()))


def make_weight_model(kind, a_dim, K, hidden_dim, num_layers):
    if kind == "mlp":
        return MLPModel(a_dim, K, hidden_dim=hidden_dim, num_layers=num_layers)
    if kind == "lstm":
        return LSTMModel(a_dim, K, hidden_dim=hidden_dim, num_layers=num_layers)
    if kind == "gated":
        return GatedModel(a_dim, K, hidden_dim=hidden_dim, num_layers=num_layers)
    raise ValueError("Invalid dynamics_parameter_network: {}".format(kind))
