"""One block of a streaming video transformer on the framework's operators: tokens of frames arrive in chunks of
any size, each chunk attends to itself and to everything before it through a key/value cache.

    python examples/streaming_block.py [--frames 6] [--height 4] [--width 6] [--chunk 17]

The block is  x += gate * Npost(attention(Npre(x)));  x += gate * Npost(mlp(Npre(x)))  with
  norms, gates and residual scale    tsn.BlockNorm: the end of one branch and the start of the next in one call
  positions (time, height, width)    tsn.RopeAxes: after the per-head norm, keys written straight into the cache
  attention                          tsn.DiffAttention: the difference of two maps, causal from the end of the cache
  projections                        Device.gemm (float32 activations, float16 weights)
Run over the same tokens in chunks of different sizes it gives the same result up to rounding; the script
prints by how much the two differ.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thinksound-native_b200"))
import tsn  # noqa: E402


class StreamingBlock:
    """A block with its cache, random weights from `seed`. `d`: width of one attention map (a head's values are 2 d)."""

    def __init__(self, dev, C=512, heads=4, kv_heads=2, d=64, axis_pairs=(8, 12, 12), batch=2, cache=512, seed=0):
        self.dev, self.C, self.H, self.Hk, self.d, self.B = dev, C, heads, kv_heads, d, batch
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        linear = lambda n, k: (r(n, k) * k ** -0.5).half()  # noqa: E731
        ones = lambda n: 1.0 + 0.1 * r(n)  # noqa: E731
        self.wq, self.wk, self.wv = linear(heads * 2 * d, C), linear(kv_heads * 2 * d, C), linear(kv_heads * 2 * d, C)
        self.wo, self.w1, self.w2 = linear(C, heads * 2 * d), linear(4 * C, C), linear(C, 4 * C)
        # the modulation of one step: shift, scale and gate of both branches, a row per sequence
        self.shift1, self.scale1, self.gate1, self.shift2, self.scale2, self.gate2 = (0.3 * r(batch, 1, C) for _ in range(6))
        self.first = tsn.BlockNorm(dev, C, post="none", pre="rms", pre_weight=ones(C))
        self.middle = tsn.BlockNorm(dev, C, post="rms", pre="rms", post_weight=ones(C), pre_weight=ones(C), residual_scale=0.9,
                                    gate_tanh=True)
        self.last = tsn.BlockNorm(dev, C, post="rms", pre="none", post_weight=ones(C), residual_scale=0.9, gate_tanh=True)
        q_norm, k_norm = ones(d), ones(d)
        self.rope = tsn.RopeAxes(dev, d, axis_pairs, q_norm=q_norm, k_norm=k_norm)
        self.rope_k = tsn.RopeAxes(dev, d, axis_pairs, k_norm=k_norm)   # an object for each place: calls of one form skip the checks
        self.attention = tsn.DiffAttention(dev, d, *(0.1 * r(d) for _ in range(4)), lambda_init=0.4, norm_weight=ones(2 * d))
        self.k_cache = torch.empty(batch, kv_heads, cache, 2 * d, dtype=torch.float16, device="cuda")   # head-major
        self.v_cache = torch.empty_like(self.k_cache)
        self.seen = 0

    def _linear(self, x, w):
        """x [B, T, K] times w [N, K] transposed, in float32."""
        y = torch.empty(*x.shape[:-1], w.shape[0], device="cuda")
        self.dev.gemm(True, w, x, y, None, x.shape[0] * x.shape[1], w.shape[0], w.shape[1])
        return y

    def __call__(self, x, pos):
        """x [B, T, C] float32, the next T tokens; pos [T, 3] int32, their time, row and column. Returns [B, T, C]."""
        B, T, C = x.shape
        d, H, Hk, at, end = self.d, self.H, self.Hk, self.seen, self.seen + T
        if end > self.k_cache.shape[2]:
            raise ValueError(f"the cache holds {self.k_cache.shape[2]} tokens")
        h, x1, x2 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        self.first(x, shift=self.shift1, scale=self.scale1, h=h)
        # a head of 2 d is two map heads of d to the rotary positions
        q = self._linear(h, self.wq).half().view(B, T, 2 * H, d)
        k = self._linear(h, self.wk).half().view(B, T, 2 * Hk, d)
        self.v_cache[:, :, at:end].copy_(self._linear(h, self.wv).view(B, T, Hk, 2 * d).transpose(1, 2))
        cached = self.k_cache[:, :, at:end].transpose(1, 2)                                    # [B, T, Hk, 2 d]
        for half in (0, 1):   # the maps' halves of the cache's heads
            self.rope_k(None, k[:, :, half::2], pos, k_out=cached[..., half * d:(half + 1) * d])
        self.rope(q, None, pos)
        o = torch.empty(B, T, H, 2 * d, dtype=torch.float16, device="cuda")
        self.attention(q.view(B, T, H, 2 * d), self.k_cache[:, :, :end].transpose(1, 2), self.v_cache[:, :, :end].transpose(1, 2), o,
                       causal=True)
        y = self._linear(o.view(B, T, -1).float(), self.wo)
        self.middle(x, y, gate=self.gate1, shift=self.shift2, scale=self.scale2, x_out=x1, h=h)
        y = self._linear(torch.nn.functional.silu(self._linear(h, self.w1)), self.w2)
        self.last(x1, y, gate=self.gate2, x_out=x2)
        self.seen = end
        return x2


def positions(frames, height, width):
    grid = torch.meshgrid(*(torch.arange(n, device="cuda") for n in (frames, height, width)), indexing="ij")
    return torch.stack(grid, -1).reshape(-1, 3).to(torch.int32).contiguous()


def run(dev, frames, height, width, chunk, seed=0):
    """The block over all tokens in chunks of `chunk`: [B, tokens, C]."""
    block = StreamingBlock(dev, cache=frames * height * width, seed=seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1)
    x, pos = torch.randn(block.B, frames * height * width, block.C, generator=g, device="cuda"), positions(frames, height, width)
    return torch.cat([block(x[:, i:i + chunk].contiguous(), pos[i:i + chunk]) for i in range(0, x.shape[1], chunk)], 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("--frames", 6), ("--height", 4), ("--width", 6), ("--chunk", 17)):
        ap.add_argument(name, type=int, default=value)
    a = ap.parse_args()
    dev = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    whole = run(dev, a.frames, a.height, a.width, a.frames * a.height * a.width)
    chunks = run(dev, a.frames, a.height, a.width, a.chunk)
    dev.commit()
    print(f"{whole.shape[1]} tokens at once and in chunks of {a.chunk}: relative difference "
          f"{float((whole - chunks).norm() / whole.norm()):.1e}")
    dev.close()


if __name__ == "__main__":
    main()
