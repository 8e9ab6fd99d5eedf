"""MLPNetwork (gfnerf/mlp.py:3-57): nn.Linear stack with bias, ReLU hidden, optional Sigmoid output; the layers run
on the f32-MFMA kernels (gfn_linear_fwd / gfn_linear_bwd) through one autograd Function per layer.

GatedMLPNetwork: the same stack with gated hidden layers (act(x Wg^T + bg) * (x Wu^T + bu), gfn_gated_fwd / gfn_gated_bwd) and dropout
behind them; no reference counterpart."""
import weakref

import torch
from torch import nn
from torch.autograd.function import once_differentiable
from torch.utils.weak import WeakIdKeyDictionary

from .. import _lib, dist, ops


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W, b, act, alive=None):
        ctx.alive = alive
        x = x.contiguous()
        y = ops.linear_fwd(x, W.contiguous(), b.contiguous(), act)
        ctx.save_for_backward(x, W, y)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, dy):
        x, W, y = ctx.saved_tensors
        dx, dW, db = ops.linear_bwd(x, W.contiguous(), y, dy.contiguous(), ctx.act, need_dx=ctx.needs_input_grad[0])
        return dx, dW, db, None, None


class MLPNetwork(nn.Module):
    def __init__(self, n_input_dims, n_output_dims, network_config, seed=1337):
        super().__init__()
        self.n_input_dims = n_input_dims
        self.n_output_dims = n_output_dims
        self.network_config = network_config
        self.n_neurons = network_config["n_neurons"]
        self.n_hidden_layers = network_config["n_hidden_layers"]
        self.sigmoid_out = network_config["output_activation"] == "Sigmoid"
        assert network_config["activation"] == "ReLU"
        self.layers = nn.ModuleList()
        for i in range(self.n_hidden_layers + 1):
            n_in = self.n_input_dims if i == 0 else self.n_neurons
            n_out = self.n_output_dims if i == self.n_hidden_layers else self.n_neurons
            self.layers.append(nn.Linear(n_in, n_out))

    def forward(self, x):
        shape = x.shape[:-1]
        x = x.reshape(-1, x.shape[-1]).float()
        for i, layer in enumerate(self.layers):
            last = i == self.n_hidden_layers
            act = ("sigmoid" if self.sigmoid_out else "none") if last else "relu"
            x = _LinearFn.apply(x, layer.weight, layer.bias, act)
        return x.reshape(*shape, -1)


class _Alive:
    """Stands for one recorded forward: it lives as long as the autograd node that holds it."""


_EAGER = WeakIdKeyDictionary()  # leaf -> its recorded forwards that are alive


def one_graph_at_a_time(*tensors):
    """What a forward of these tensors holds on to while its autograd graph lives (None: nothing is recorded).  Refuses to
    record a forward into a hipGraph while an eager autograd graph of the same leaves lives.  The leaf's gradient accumulator
    belongs to that graph and to its stream; a captured backward would wait for a stream outside the capture, and ending the capture then ends
    the process.  Drop the eager outputs (or detach them) before capturing.  Of leaves that a caller's own operations stand in front of nothing is
    known here."""
    leaves = [t for t in tensors if t is not None and t.requires_grad and t.is_leaf] if torch.is_grad_enabled() else []
    if not leaves:
        return None
    if torch.cuda.is_current_stream_capturing():
        for t in leaves:
            if len(_EAGER.get(t, ())):
                raise _lib.GfnError("a forward of these parameters is being captured while an eager autograd graph of them is alive: drop its outputs first")
        return None
    alive = _Alive()
    for t in leaves:
        _EAGER.setdefault(t, weakref.WeakSet()).add(alive)
    return alive


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, Wg, Wu, bg, bu, act, alive):
        Wg, Wu, bg, bu = (t if t is None else t.contiguous() for t in (Wg, Wu, bg, bu))
        h = ops.gated_fwd(x, Wg, Wu, bg, bu, act)
        ctx.save_for_backward(x, Wg, Wu, bg, bu)
        ctx.act, ctx.alive = act, alive
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, Wg, Wu, bg, bu = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dWg, dWu, dbg, dbu = ops.gated_bwd(x, Wg, Wu, dh.contiguous(), bg, bu, ctx.act, need_dx=need[0], need_dw=any(need[1:5]))
        return dx, dWg, dWu, dbg, dbu, None, None


def gated_linear(x, Wg, Wu, bg=None, bu=None, act="silu"):
    """act(x Wg^T + bg) * (x Wu^T + bu) over the last dimension of x, with gradients (ops.gated_fwd / ops.gated_bwd)."""
    alive = one_graph_at_a_time(x, Wg, Wu, bg, bu)
    return _GatedFn.apply(x.reshape(-1, x.shape[-1]).contiguous(), Wg, Wu, bg, bu, act, alive).reshape(*x.shape[:-1], Wg.shape[0])


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, call, alive):
        ctx.p, ctx.seed, ctx.call, ctx.alive = p, seed, call, alive
        return ops.dropout(x, p, seed, call)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return ops.dropout(dy.contiguous(), ctx.p, ctx.seed, ctx.call), None, None, None, None


class Dropout(nn.Module):
    """Dropout over the last dimension with a mask that is never stored (ops.dropout): a function of the module's seed, the number of its
    forward passes in training mode (`counter`, on the device: replayed graphs draw fresh masks), the row and the column.  Every forward pass
    draws a mask of its own, so one that is run again inside a backward pass is refused.  seed: default, a number from torch's generator
    (torch.manual_seed), so that modules differ; a copy of a module draws the module's masks.  The ranks of a distributed run differ whatever
    the seed."""

    def __init__(self, p: float = 0.5, seed=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p = {p} is not in [0, 1]")
        self.p, self.seed = float(p), int(torch.randint(1 << 62, (), device="cpu")) if seed is None else int(seed)
        self.register_buffer("counter", torch.zeros(1, dtype=torch.int64))

    def key(self):
        """The masks' key on this rank (rank 0, and without a process group: the seed)."""
        return (self.seed + dist.rank() * 0x9E3779B97F4A7C15) & 0xFFFFFFFFFFFFFFFF

    def forward(self, x):
        if not self.training or self.p == 0.0 or 0 in x.shape[-1:]:
            return x
        if torch._C._current_graph_task_id() != -1:
            raise _lib.GfnError("a dropout is recomputed inside a backward pass (torch.utils.checkpoint): it would draw another mask than its first forward; "
                                "leave it outside of the recomputed part (it keeps nothing of its input)")
        alive = one_graph_at_a_time(x)
        return _DropoutFn.apply(x.reshape(-1, x.shape[-1]).contiguous(), self.p, self.key(), ops.dropout_call(self.counter), alive).reshape(x.shape)


class GatedLayer(nn.Module):
    """One gated hidden layer: `gate` and `up` are nn.Linear parameter holders (the kernels read their tensors)."""

    def __init__(self, n_in, n_out, act):
        super().__init__()
        self.gate, self.up, self.act = nn.Linear(n_in, n_out), nn.Linear(n_in, n_out), act

    def forward(self, x):
        return gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, self.act)


class GatedMLPNetwork(nn.Module):
    """MLPNetwork's arguments and call with gated hidden layers: network_config["activation"] is "SwiGLU", "GEGLU", "ReGLU" or "GLU";
    network_config["dropout"] (default 0) is applied behind every hidden layer in training mode, with seeds seed, seed + 1, .. (default: Dropout's).  Computes in f32 like MLPNetwork;
    at most 128 inputs and 128 neurons (the layers' kernels)."""

    ACTIVATIONS = {"SwiGLU": "silu", "GEGLU": "gelu", "ReGLU": "relu", "GLU": "sigmoid"}

    def __init__(self, n_input_dims, n_output_dims, network_config, seed=None):
        super().__init__()
        if network_config["activation"] not in self.ACTIVATIONS:
            raise ValueError(f"activation {network_config['activation']!r} is none of {sorted(self.ACTIVATIONS)}")
        self.n_input_dims, self.n_output_dims, self.network_config = n_input_dims, n_output_dims, network_config
        self.n_neurons, self.n_hidden_layers = network_config["n_neurons"], network_config["n_hidden_layers"]
        self.sigmoid_out = network_config["output_activation"] == "Sigmoid"
        act = self.ACTIVATIONS[network_config["activation"]]
        widths = [n_input_dims] + [self.n_neurons] * self.n_hidden_layers
        self.layers = nn.ModuleList(GatedLayer(a, b, act) for a, b in zip(widths, widths[1:]))
        self.layers.append(nn.Linear(widths[-1], n_output_dims))
        p = float(network_config.get("dropout", 0.0))
        self.dropout = nn.ModuleList(Dropout(p, None if seed is None else seed + i) for i in range(self.n_hidden_layers)) if p else None

    def forward(self, x):
        out, shape = self.layers[-1], x.shape[:-1]
        alive = one_graph_at_a_time(x, out.weight, out.bias)  # the hidden layers see to their own
        x = x.reshape(-1, x.shape[-1]).float()
        for i in range(self.n_hidden_layers):
            x = self.layers[i](x)
            if self.dropout is not None:
                x = self.dropout[i](x)
        return _LinearFn.apply(x, out.weight, out.bias, "sigmoid" if self.sigmoid_out else "none", alive).reshape(*shape, -1)
