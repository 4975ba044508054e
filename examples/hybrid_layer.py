"""A layer with two memories on the same tokens: the recurrent state of the GDN3 scan, which carries the whole
past, and exact attention over a sliding window and the first tokens, which carries the recent past.

    python examples/hybrid_layer.py

runs, on synthetic projections, what a model does with it: a training step, a batch of prompts, samples forked
from them that share the prompts' pages, steps of one token each, and closing the cache's pool up.  Every token
that the decode produces is checked against the prompt path over the same sequence.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from gdnx_b200 import ops  # noqa: E402


class HybridLayer:
    """H scan heads of M lanes beside H query heads on Hk key heads, all of size D.  The scan's state [slots*H*M, D, D]
    and the cache's slots belong together: slot s is one sequence in both."""

    def __init__(self, H=4, Hk=2, M=4, D=128, window=64, sinks=4, *, slots=8, pages=64, page=16, dtype=torch.bfloat16,
                 device="cuda"):
        self.H, self.Hk, self.M, self.D, self.window, self.sinks = H, Hk, M, D, window, sinks
        self.cache = ops.PagedCache.zeros(1, pages, Hk, page, D, slots=slots, width=pages, dtype=dtype, device=device)
        self.state = torch.zeros(slots, H * M, D, D, device=device)

    def mix(self, y_scan, y_attn):
        """The lanes' mean beside the exact read."""
        return y_scan.float().mean(-2) + y_attn.float()

    def train(self, t):
        """Both memories of whole sequences, differentiable in every projection."""
        y_scan, _ = ops.gdn3_scan_train(t["q"], t["ks"], t["vs"], t["beta"], t["beta"], t["logg"], decay_kind="log")
        y_attn = ops.window_attention_train(t["q"], t["k"], t["v"], window=self.window, sinks=self.sinks)
        return self.mix(y_scan, y_attn)

    def prompt(self, t, slots):
        """The prompts `t` [B,T,...] into the free slots `slots` (int32): outputs [B,T,H,D]."""
        B, T = t["k"].shape[:2]
        y_scan, state = ops.gdn3_scan(t["q"], t["ks"], t["vs"], t["beta"], t["beta"], t["logg"], decay_kind="log",
                                      return_state=True)
        self.state[slots.long()] = state.view(B, -1, self.D, self.D)
        ops.cache_extend(self.cache, slots, torch.full_like(slots, T))
        ops.cache_write(self.cache, t["k"], t["v"], slots)
        ops.cache_trim(self.cache, slots, window=self.window, sinks=self.sinks)
        return self.mix(y_scan, ops.window_attention(t["q"], t["k"], t["v"], window=self.window, sinks=self.sinks))

    def fork(self, src, dst):
        """Slots `dst` become samples of `src`: the state is copied, the pages are shared until written."""
        self.state[dst.long()] = self.state[src.long()]
        ops.cache_fork(self.cache, src, dst)

    def step(self, t, slots):
        """One token `t` [B,1,...] for each of `slots`: outputs [B,H,D]."""
        state = self.state[slots.long()].flatten(0, 1)
        one = {n: x[:, 0] for n, x in t.items()}
        y_scan = ops.decode_step(state, one["q"], one["ks"], one["vs"], one["beta"], one["beta"], one["logg"],
                                 decay_kind="log")
        self.state[slots.long()] = state.view(slots.shape[0], -1, self.D, self.D)
        ops.cache_extend(self.cache, slots, torch.ones_like(slots))
        ops.cache_write(self.cache, t["k"], t["v"], slots)
        y_attn = ops.paged_decode(one["q"], self.cache, rows=slots, window=self.window, sinks=self.sinks)
        ops.cache_trim(self.cache, slots, window=self.window, sinks=self.sinks)
        return self.mix(y_scan, y_attn)

    def drop(self, slots):
        """Frees slots and moves the remaining pages together."""
        ops.cache_truncate(self.cache, slots, torch.zeros_like(slots))
        ops.cache_compact(self.cache)


def projections(layer, B, T, seed, dtype=torch.bfloat16, device="cuda"):
    """Synthetic projections: unit keys and queries for the scan, gates and decays as the layer makes them."""
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    unit = lambda x: torch.nn.functional.normalize(x, dim=-1)  # noqa: E731
    H, Hk, M, D = layer.H, layer.Hk, layer.M, layer.D
    t = dict(q=unit(r(B, T, H, D)) * 4, ks=unit(r(B, T, H, D)), vs=r(B, T, H, D), k=r(B, T, Hk, D), v=r(B, T, Hk, D),
             beta=torch.sigmoid(r(B, T, H, M)), logg=-torch.nn.functional.softplus(r(B, T, H, M) - 3))
    return {n: x.to(dtype if n not in ("logg",) else torch.float32) for n, x in t.items()}


def join(a, b):
    return {n: torch.cat([a[n], b[n]], 1) for n in a}


def main(steps=6, T=150):
    layer = HybridLayer()
    dev = layer.state.device
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731

    t = {n: x.requires_grad_() for n, x in projections(layer, 2, 96, 1).items()}
    layer.train(t).square().mean().backward()
    grads = {n: x.grad.float().norm().item() for n, x in t.items()}

    prompts = projections(layer, 2, T, 2)
    layer.prompt(prompts, i32(0, 1))
    layer.fork(i32(0, 0, 1), i32(2, 3, 4))  # two samples of the first prompt, one of the second
    slots, of = i32(0, 1, 2, 3, 4), [0, 1, 0, 0, 1]
    seen, worst = {n: x[of] for n, x in prompts.items()}, 0.0
    for n in range(steps):
        token = projections(layer, 5, 1, 10 + n)
        seen = join(seen, token)
        y = layer.step(token, slots)
        whole = HybridLayer(slots=5, pages=64).prompt(seen, i32(0, 1, 2, 3, 4))[:, -1]
        worst = max(worst, ((y - whole).norm() / whole.norm()).item())
    layer.drop(i32(1, 3))
    ops.cache_check(layer.cache)  # no operation was refused
    ops.check_device_status()
    live = int((layer.cache.refs > 0).sum())
    assert bool((layer.cache.refs[:live] > 0).all())
    return dict(grads=grads, worst=worst, live=live)


if __name__ == "__main__":
    r = main()
    print("gradient norms: " + ", ".join("%s %.3g" % x for x in r["grads"].items()))
    print("decode against the prompt path: relative difference %.2g; %d live pages, at the pool's start" % (r["worst"], r["live"]))
