"""Channels-last building blocks shared by every model family.

All spatial activations are ``[B, H, W, C]`` and all token activations
``[B, N, C]``; every heavy op goes through ``arbius_amd.ops`` (HIP kernels on
GPU, PyTorch reference on CPU).  Parameters are plain tensors registered on
``nn.Module`` so weights can be RCCL-broadcast / loaded from safetensors
without any framework glue.

Random init is deterministic per module path (``init_weights(seed)``): the
benchmark runs random-init weights of the real architectures.
"""
from __future__ import annotations

import math
import threading

import torch
import torch.nn as nn

from .. import ops

# Captures are serialised process-wide; "thread_local" capture mode lets other threads keep
# launching work on their own streams while one thread captures (concurrent task streams).
CAPTURE_LOCK = threading.RLock()
_USES = threading.local()        # .log: the Int8Uses entered on this thread
_SWITCHES = [None]               # another object after every change of a layer between 16 and 8 bits


class Int8Uses:
    """``with Int8Uses() as uses:`` - the form (``Int8Rows``, or None: 16 bits) of every ``Linear`` that this thread
    runs meanwhile.  A captured graph keeps one: it holds the 8-bit tensors whose addresses the graph replays, and
    ``current`` tells whether they still are what the layers would run on."""

    def __init__(self):
        self.forms, self.weights, self.seen = {}, (), _SWITCHES[0]

    def __enter__(self):
        self.prev, _USES.log = getattr(_USES, "log", None), self.forms
        return self

    def __exit__(self, *exc):
        _USES.log = self.prev
        self.weights = [(lin._parameters, lin._parameters["weight"], *lin._of[:2])
                        for lin, form in self.forms.values() if form is not None and form is lin.int8]

    def current(self) -> bool:
        switches = _SWITCHES[0]
        if switches is not self.seen:
            if any(lin.int8 is not form for lin, form in self.forms.values()):
                return False
            self.seen = switches
        for params, w, ptr, version in self.weights:               # as Linear.outdated, before every replay
            if w._version != version or w.data_ptr() != ptr or params["weight"] is not w:
                return False
        return True


class Linear(nn.Module):
    """``hoisted``: never called itself, its bare weight is read as a part of a batched projection (so it has no 8-bit
    form)."""

    def __init__(self, cin, cout, bias=True, hoisted=False):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(cout, cin), requires_grad=False)
        self.bias = nn.Parameter(torch.empty(cout), requires_grad=False) if bias else None
        self.cin, self.cout, self.hoisted = cin, cout, hoisted
        self.int8 = None              # ops.Int8Rows of the weight: this linear runs in 8 bits (int8_linears)

    @property
    def int8(self):
        return self._int8

    @int8.setter
    def int8(self, rows):
        self._int8, self._of = rows, None if rows is None else self._weight()
        _SWITCHES[0] = object()

    def _weight(self):
        w = self._parameters["weight"]
        return w.data_ptr(), w._version, w.dtype

    def reset(self, gen):
        bound = 1.0 / math.sqrt(self.cin)
        self.weight.data.uniform_(-bound, bound, generator=gen)
        if self.bias is not None:
            self.bias.data.uniform_(-bound, bound, generator=gen)

    def outdated(self) -> bool:
        """Whether the weight holds other values than its 8-bit form was made of."""
        return self._of != self._weight()

    def form(self):
        """The ``Int8Rows`` this layer runs on, None in 16 bits; noted for the capture under way on this thread."""
        int8, log = self._int8, getattr(_USES, "log", None)
        if int8 is not None and self.outdated():
            with CAPTURE_LOCK:                                     # forks come here at once: one of them quantises
                if self.outdated():
                    _publish([self], [ops.quantize_rows(self.weight)])
                int8 = self._int8
        if log is not None:
            log[id(self), id(int8)] = self, int8
        return int8

    def forward(self, x, residual=None, act=None):
        int8 = self.form()
        if int8 is not None:
            return ops.linear_int8(x, int8, self.bias, residual=residual, act=act)
        return ops.linear(x, self.weight, self.bias, residual=residual, act=act)

    def forward_norm(self, x, norm):
        """x [B, ..., Cin] with a GroupNorm(+SiLU) prologue from ``norm = (table, silu)`` (table per
        batch row b): run as a 1x1 implicit-GEMM conv over the [B, 1, N, Cin] view (8 bits: in a pass of its own)."""
        int8 = self.form()
        if int8 is not None:
            return ops.linear_int8(ops.normed(x, norm), int8, self.bias)
        B, C = x.shape[0], x.shape[-1]
        y = ops.conv2d(x.reshape(B, 1, -1, C), self.weight.view(self.cout, 1, 1, self.cin), self.bias,
                       padding=0, norm=norm)
        return y.view(*x.shape[:-1], self.cout)

    def geglu(self, x):
        """GEGLU projection (ops.linear_geglu)."""
        int8 = self.form()
        if int8 is not None:
            return ops.linear_int8(x, int8, self.bias, act="geglu")
        return ops.linear_geglu(x, self.weight, self.bias)


class Conv2d(nn.Module):
    """kxk conv, stride 1 or 2, channels-last; weight [Cout, k, k, Cin]."""

    def __init__(self, cin, cout, k=3, stride=1, padding=None, bias=True):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(cout, k, k, cin), requires_grad=False)
        self.bias = nn.Parameter(torch.empty(cout), requires_grad=False) if bias else None
        self.cin, self.cout, self.k, self.stride = cin, cout, k, stride
        self.padding = k // 2 if padding is None else padding

    def reset(self, gen):
        bound = 1.0 / math.sqrt(self.cin * self.k * self.k)
        self.weight.data.uniform_(-bound, bound, generator=gen)
        if self.bias is not None:
            self.bias.data.uniform_(-bound, bound, generator=gen)

    def forward(self, x, upsample=False, residual=None, temb=None, norm=None):
        """``norm = (table, silu)``: GroupNorm(+SiLU) prologue fused into the conv."""
        return ops.conv2d(x, self.weight, self.bias, stride=self.stride, padding=self.padding,
                          upsample=upsample, residual=residual, temb=temb, norm=norm)


class GroupNorm(nn.Module):
    def __init__(self, groups, channels, eps=1e-5, silu=False):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(channels), requires_grad=False)
        self.bias = nn.Parameter(torch.zeros(channels), requires_grad=False)
        self.groups, self.eps, self.silu = groups, eps, silu

    def reset(self, gen):
        self.weight.data.fill_(1.0)
        self.bias.data.zero_()

    def forward(self, x, silu=None):
        return ops.group_norm(x, self.weight, self.bias, self.groups, self.eps,
                              self.silu if silu is None else silu)

    def table(self, x, mod=None, one_plus=0.0, silu=None):
        """This GroupNorm of ``x`` for a consumer (``ops.NormSpec``): a fused operand prologue from
        the (lazily computed) affine table, or one stats + table-apply pass in front of it."""
        return ops.NormSpec(x, self.weight, self.bias, self.groups, self.eps, mod, one_plus,
                            self.silu if silu is None else silu)


class LayerNorm(nn.Module):
    def __init__(self, channels, eps=1e-5):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(channels), requires_grad=False)
        self.bias = nn.Parameter(torch.zeros(channels), requires_grad=False)
        self.eps = eps

    def reset(self, gen):
        self.weight.data.fill_(1.0)
        self.bias.data.zero_()

    def forward(self, x):
        return ops.layer_norm(x, self.weight, self.bias, self.eps)

    def linear(self, x, lin: "Linear", residual=None, act=None):
        """act(lin(self(x))) with this LayerNorm (and the activation) folded into the GEMM (ops.ln_linear)."""
        int8 = lin.form()
        if int8 is not None:
            return ops.ln_linear_int8(x, self.weight, self.bias, self.eps, int8, lin.bias, residual=residual, act=act)
        return ops.ln_linear(x, self.weight, self.bias, self.eps, lin.weight, lin.bias, residual=residual, act=act)

    def linear_geglu(self, x, lin: "Linear"):
        """GEGLU projection of self(x) with this LayerNorm folded in (ops.ln_linear_geglu)."""
        int8 = lin.form()
        if int8 is not None:
            return ops.ln_linear_int8(x, self.weight, self.bias, self.eps, int8, lin.bias, act="geglu")
        return ops.ln_linear_geglu(x, self.weight, self.bias, self.eps, lin.weight, lin.bias)


class Embedding(nn.Module):
    def __init__(self, n, dim):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(n, dim), requires_grad=False)

    def reset(self, gen):
        self.weight.data.normal_(0.0, 0.02, generator=gen)

    def forward(self, idx):
        return self.weight[idx]


def init_weights(module: nn.Module, seed: int = 0) -> nn.Module:
    """Deterministic random init of every leaf with a ``reset(gen)``, in
    module-registration order, from one CPU generator."""
    gen = torch.Generator(device="cpu").manual_seed(seed)
    for m in module.modules():
        if hasattr(m, "reset") and m is not module:
            m.reset(gen)
    return module


def packed_positions(ids, offsets, longest):
    """Of every token of prompts packed end to end (offsets int32 [n + 1], the prompts' first tokens and the end): its
    position in its prompt, and whether it is outside - of every prompt, or past the ``longest`` tokens a model
    has positions for (the position is clamped then; nothing here waits for the device)."""
    at = torch.arange(ids.shape[0], device=ids.device, dtype=torch.int32)
    doc = torch.searchsorted(offsets, at, right=True) - 1
    pos = at - offsets[doc]
    outside = (doc < 0) | (doc >= offsets.shape[0] - 1) | (pos < 0) | (pos >= longest)
    return pos.clamp(0, longest - 1), outside


def int8_linears(module: nn.Module, on: bool = True) -> int:
    """Run the ``Linear`` layers of ``module`` in 8 bits (``ops.linear_int8``; weights quantised here, once, per output
    channel; activations per token as they come) or, with ``on=False``, in their own type again.  An
    operator's choice per deployment: other bytes than the 16-bit layers, so never for a registered model
    whose solutions other nodes verify.  Returns the number of layers; ``hoisted`` ones, of which only the bare
    weight is used, stay in 16 bits and are not counted.  Weights loaded or moved later are quantised again at their
    next use (changed through ``.data``, which torch does not count, only by another call).

    All weights are quantised before the first layer changes, and their kernels have finished: pipeline forks share
    the layers across threads and streams (``ops.derived_ready``).  Pipelines capture their graphs again at their next
    call, after this one and after a change of weights.  Call it while none is solving: 8-bit weights that it replaces
    are given back once what the GPUs were doing is done."""
    linears = [m for m in module.modules() if isinstance(m, Linear) and not m.hoisted]
    _publish(linears, [ops.quantize_rows(m.weight) if on else None for m in linears])
    return len(linears)


def _publish(linears, forms):
    """Give the layers these 8-bit forms (or None) once the kernels that write them have finished, and give the old ones
    back once the kernels of any stream that read them have."""
    for q in {f.device: f.q for f in forms if f is not None}.values():
        ops.derived_ready(q)
    old = {}
    for m, form in zip(linears, forms):
        if m.int8 is not None:
            old.setdefault(m.int8.device, []).append(m.int8)
        m.int8 = form
    for device in old:
        if device.type == "cuda":
            with CAPTURE_LOCK:         # a device is not waited for while a thread captures on it
                torch.cuda.synchronize(device)


def timestep_embedding(t, dim, flip_sin_to_cos=True, freq_shift=0.0, max_period=10000):
    """Sinusoidal timestep features (diffusers ``get_timestep_embedding`` semantics)."""
    half = dim // 2
    exponent = -math.log(max_period) * torch.arange(half, dtype=torch.float32, device=t.device)
    exponent = exponent / (half - freq_shift)
    emb = t.float()[:, None] * torch.exp(exponent)[None, :]
    emb = torch.cat([torch.sin(emb), torch.cos(emb)], dim=-1)
    if flip_sin_to_cos:
        emb = torch.cat([emb[:, half:], emb[:, :half]], dim=-1)
    return emb


def fuse_qkv(layers):
    """Concatenate the weights of several bias-free Linear layers into one GEMM."""
    return torch.cat([l.weight for l in layers], dim=0)
