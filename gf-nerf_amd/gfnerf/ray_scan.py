"""Recurrences along the packed samples of rays (ops.ray_scan_fwd / ray_scan_bwd / ray_scan_step): the autograd function, a learnt gated
recurrence, and the composite of any number of feature channels -- what nerfstudio/model_components/renderers.py:69-138 does for colour.
The recurrences with learnt gates have no reference counterpart."""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .. import ops
from .mlp import _LinearFn, one_graph_at_a_time


class _RayScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pts_offsets, f, c, h0, gate, reverse, save, alive):
        r = ops.ray_scan_fwd(pts_offsets, f, c, gate, reverse, h0, save=save)
        ctx.save_for_backward(pts_offsets, f, c, h0, r["saved"])
        ctx.gate, ctx.reverse, ctx.alive = gate, reverse, alive
        ctx.set_materialize_grads(False)
        return r["h"], r["state"]

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, d_state):
        pts_offsets, f, c, h0, saved = ctx.saved_tensors
        dh = torch.zeros_like(c) if dh is None else dh.contiguous()
        g = ops.ray_scan_bwd(pts_offsets, f, c, dh, saved, ctx.gate, ctx.reverse, h0, None if d_state is None else d_state.contiguous())
        return None, g["df"], g["dc"], g["dh0"] if h0 is not None else None, None, None, None, None


def ray_scan(pts_offsets, f, c, gate="sigmoid", reverse=False, h0=None, leaves=()):
    """ops.ray_scan_fwd with gradients for f, c and h0 -> (h [n, channels], state f32 [rays, channels]).  leaves: the tensors that f and c were
    made from, where nothing else keeps a capture of this forward apart from an eager graph of theirs (one_graph_at_a_time)."""
    alive = one_graph_at_a_time(f, c, h0, *leaves)
    save = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (f, c, h0))
    return _RayScanFn.apply(pts_offsets, f.contiguous(), c.contiguous(), None if h0 is None else h0.contiguous(), gate, bool(reverse), save, alive)


def render_features(pts_offsets, sigma, dt, features):
    """Composite `features` [n, channels] along each ray with the weights T_i alpha_i, alpha = 1 - exp(-sigma dt) (RaySamples.get_weights_f2nerf,
    nerfstudio/cameras/rays.py:178-200) -> f32 [rays, channels]; gradients for sigma, dt and features.  The sum over a ray is the recurrence
    h = exp(-sigma dt) h + alpha c taken back to front: no weights array, any number of channels.  All of it is in f32 whatever the features'
    dtype (the recurrence takes its gates and inputs in one type, and a sigma dt of 16 bits would be off by 2^-9 of itself in every factor of the
    transmittance): features of 16 bits are cast."""
    thickness = sigma.reshape(-1).float() * dt.reshape(-1).float()
    return ray_scan(pts_offsets, thickness[:, None], features.float(), "decay", reverse=True, leaves=(sigma, dt, features))[1]


class RayRecurrence(nn.Module):
    """h_t = s(x_t Wf + bf) h_{t-1} + (1 - s(x_t Wf + bf)) (x_t Wc + bc) along each ray: a per-ray sequence layer whose state is `dim` wide.
    `reverse`: back to front.  forward() takes all samples of a batch of rays, step() one more sample of each."""

    def __init__(self, n_input_dims, dim, reverse=False):
        super().__init__()
        self.gate, self.input, self.reverse = nn.Linear(n_input_dims, dim), nn.Linear(n_input_dims, dim), bool(reverse)
        nn.init.constant_(self.gate.bias, 2.0)  # remembers about ten samples at the start

    def _project(self, x):
        x = x.float()
        return (_LinearFn.apply(x, layer.weight, layer.bias, "none") for layer in (self.gate, self.input))

    def forward(self, x, pts_offsets, state=None):
        """x [n, n_input_dims] packed -> (h [n, dim], state [rays, dim]); state: the rays' states in front of x (default 0)."""
        f, c = self._project(x)
        return ray_scan(pts_offsets, f, c, "sigmoid", self.reverse, state, (x, *self.parameters()))

    @torch.no_grad()
    def step(self, x, state):
        """x [rays, n_input_dims]: one more sample of every ray; state f32 [rays, dim] is advanced in place -> h [rays, dim]."""
        if self.reverse:
            raise ValueError("a back-to-front recurrence has no next sample")
        f, c = self._project(x)
        return ops.ray_scan_step(f, c, state, "sigmoid")
