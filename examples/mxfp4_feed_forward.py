"""A decoder layer's feed-forward on MXFP4 weights that come out of a compressed buffer.

The weights are coded (codes by the nibble chain, block scales by the passthrough chain), restored into HBM by one
decode call, and used where they were restored: norm with the residual's addition, product, gated activation, product.
What goes from one operator to the next in 8 bits is e4m3 codes with a scale for every 32.

    python examples/mxfp4_feed_forward.py [--hidden 4096] [--inner 14336] [--tokens 1 16 2048]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ptwm_amd import api, ids, plan  # noqa: E402

DEVICE = "cuda:0"
F8, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise_weights(w):
    """(codes, scales) of float32 weights: a block's scale leaves its largest magnitude in [4, 8), cut at 6."""
    b = w.reshape(w.shape[0], -1, 32)
    e = (torch.frexp(b.abs().amax(-1))[1] - 3).clamp(-127, 127)
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    code = torch.bucketize(torch.ldexp(b.abs(), -e.unsqueeze(-1)), bounds, out_int32=True) + 8 * (b < 0)
    code = code.to(torch.uint8).reshape(w.shape)
    return code[:, 0::2] | code[:, 1::2] << 4, (e + 127).to(torch.uint8)


def dequantise_weights(codes, scales):
    value = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = torch.stack((value[(codes & 15).int()], value[(codes >> 4).int()]), -1).reshape(codes.shape[0], -1, 32)
    return (v * scales.view(E8M0).float().unsqueeze(-1)).reshape(codes.shape[0], -1)


def compress(tensors):
    """One buffer of encoded planes and the plan that restores (codes, scales, ...) back to back."""
    chains = [plan.CHAIN_NIBBLE_SPLIT, plan.CHAIN_PASSTHROUGH] * (len(tensors) // 2)
    items = [(c, t.contiguous().view(-1)) for c, t in zip(chains, tensors)]
    out = torch.empty(sum(t.numel() for _, t in items) * 17 // 16 + 65536 * len(items), dtype=torch.uint8,
                      device=DEVICE)
    used, state = api.encode_tensors_cuda(items, out, 0)
    return out[:used].clone(), state


def restore(planes, state, shapes):
    """The tensors of the plan as views of one buffer, in the order in which they were given."""
    tensors = plan.decode_plan(state)
    out = torch.empty(tensors[-1].out_offset + tensors[-1].out_len, dtype=torch.uint8, device=DEVICE)
    api.hardware_backend_dispatch_decode_cuda(ids.HARDWARE_BACKEND_LABEL, ids.DECODE_PLAN_LABEL, state, planes, out, 0)
    return [out[t.out_offset:t.out_offset + t.out_len].view(shape) for t, shape in zip(tensors, shapes)]


class FeedForward:
    """Workspaces for up to `tokens` tokens are kept; a call works in their first rows."""

    def __init__(self, norm, gate_up, gate_up_scales, down, down_scales, tokens, eps=1e-5):
        self.norm, self.eps = norm, eps
        self.gate_up, self.gate_up_scales, self.down, self.down_scales = gate_up, gate_up_scales, down, down_scales
        hidden, inner = norm.numel(), gate_up.shape[0] // 2
        new = lambda cols, dtype: torch.empty((tokens, cols), dtype=dtype, device=DEVICE)  # noqa: E731
        self.codes, self.scales = new(hidden, F8), new(hidden // 32, E8M0)
        self.both = new(2 * inner, torch.bfloat16)
        self.act, self.act_scales = new(inner, F8), new(inner // 32, E8M0)
        self.out = new(hidden, torch.bfloat16)

    def __call__(self, x, residual):
        """The block's output for x (rows of bfloat16); residual becomes residual + x."""
        t, inner = x.shape[0], self.act.shape[1]
        codes, scales, both, out = self.codes[:t], self.scales[:t], self.both[:t], self.out[:t]
        act, act_scales = self.act[:t], self.act_scales[:t]
        api.rms_norm_mx_cuda(x, self.norm, codes, scales, 0, residual=residual, sum_out=residual, eps=self.eps)
        api.mxfp4_linear_cuda(codes, self.gate_up, self.gate_up_scales, both, 0, x_scales=scales)
        api.swiglu_mx_cuda(both[:, :inner], both[:, inner:], act, act_scales)
        api.mxfp4_linear_cuda(act, self.down, self.down_scales, out, 0, x_scales=act_scales)
        return out


def plain(x, residual, norm, gate_up, down, eps=1e-5):
    """The same block in float32, activations not rounded on the way."""
    s = x.float() + residual.float()
    y = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * norm.float()
    gate, up = (y @ gate_up.t()).chunk(2, -1)
    return (gate / (1 + torch.exp(-gate)) * up) @ down.t(), s


def main(hidden=4096, inner=14336, tokens=(1, 16, 2048), seed=0):
    """Prints what it does; returns the largest relative error of the block's output."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    made = [*quantise_weights(normal(2 * inner, hidden) * 0.02), *quantise_weights(normal(hidden, inner) * 0.02)]
    planes, state = compress(made)
    raw = sum(t.numel() for t in made)
    back = restore(planes, state, [t.shape for t in made])
    assert all(torch.equal(a, b) for a, b in zip(made, back)), "the restored weights differ"
    print(f"weights {raw} bytes, compressed {planes.numel()}, restored exactly")
    norm = (1 + 0.1 * normal(hidden)).to(torch.bfloat16)
    block = FeedForward(norm, *back, max(tokens))
    dense = dequantise_weights(*made[:2]), dequantise_weights(*made[2:])
    worst = 0.0
    for t in tokens:
        x, residual = normal(t, hidden).to(torch.bfloat16), (4 * normal(t, hidden)).to(torch.bfloat16)
        want, total = plain(x, residual, norm, *dense)
        stream = residual.clone()
        got = block(x, stream).float()
        error = ((got - want).norm() / want.norm()).item()
        assert torch.equal(stream, total.to(torch.bfloat16)), "the residual stream differs"
        worst = max(worst, error)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(20):
            block(x, stream)
        end.record()
        end.synchronize()
        print(f"{t:5d} tokens: {start.elapsed_time(end) / 20 * 1e3:8.1f} us, relative error {error:.4f}")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--inner", type=int, default=14336)
    ap.add_argument("--tokens", type=int, nargs="+", default=[1, 16, 2048])
    a = ap.parse_args()
    main(a.hidden, a.inner, a.tokens)
