"""Frames of an online reconstruction through a small transformer on the token operators.

Each new frame (512 x 384 pixels, 768 tokens of 16 x 16 patches) goes through blocks that

  * place queries and keys by patch row and column (``Rotary``, two axes),
  * keep the frame's keys and values in 8 bits, 12 blocks of 64 tokens (``KVCache.append``),
  * look at the frame itself and at the kept frames most like it (``KVCache.attend`` over a list of their blocks),

and a head turns the tokens into the log-depth channels that bundle adjustment samples at its keypoints
(``sample_depth_maps``).  The weights are random, so the depths mean nothing; what is printed is the cache's size and how far
the 8-bit attention of the last frame is from attention over the unrounded keys and values.

    python examples/online_frames.py --frames 8 --layers 2
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from blast3r_amd.kv_cache import BLOCK, KVCache  # noqa: E402
from blast3r_amd.rotary import Rotary  # noqa: E402
from blast3r_amd.sampling import sample_depth_maps  # noqa: E402

PATCH, ROWS, COLS = 16, 24, 32
TOKENS = ROWS * COLS
FRAME_BLOCKS = TOKENS // BLOCK


class Layer:
    """One attention block with its cache of all frames."""

    def __init__(self, width, heads, frames, bits, rotary, gen, dev):
        self.heads, self.dim, self.rotary = heads, width // heads, rotary

        def weight(n, m):
            return (torch.randn((n, m), generator=gen, device=dev) / math.sqrt(m)).bfloat16()

        self.qkv, self.out = weight(3 * width, width), weight(width, width)
        self.up, self.down = weight(4 * width, width), weight(width, 4 * width)
        self.cache = KVCache(frames * FRAME_BLOCKS, heads, self.dim, bits, device=dev)

    def __call__(self, x, positions, own, seen, lengths):
        """x (768, width); own: the frame's blocks, seen: the blocks looked at, its own last."""
        h = torch.nn.functional.layer_norm(x, x.shape[-1:])
        qkv = (h @ self.qkv.t()).view(TOKENS, 3 * self.heads, self.dim)
        q, k = self.rotary(positions, qkv[:, :self.heads], qkv[:, self.heads:2 * self.heads])
        v = qkv[:, 2 * self.heads:]
        self.cache.append(k, v, own, torch.zeros_like(lengths))
        o = self.cache.attend(q, seen, lengths, causal=False)
        x = x + o.reshape(TOKENS, -1) @ self.out.t()
        h = torch.nn.functional.layer_norm(x, x.shape[-1:])
        return x + torch.nn.functional.gelu(h @ self.up.t()) @ self.down.t(), (q, k, v, o)


def plain_attention(q, k, v):
    """softmax(q k^T / sqrt(dim)) v of (tokens, heads, dim) tensors in fp32."""
    q, k, v = (t.float().transpose(0, 1) for t in (q, k, v))
    p = torch.softmax(torch.matmul(q, k.transpose(1, 2)) / math.sqrt(q.shape[-1]), -1)
    return torch.matmul(p, v).transpose(0, 1)


@torch.no_grad()
def run(frames=8, layers=2, width=1024, heads=16, like=4, channels=5, bits=torch.float8_e4m3fn, seed=0, device='cuda'):
    """Returns (relative error of the last frame's attention in the first layer, the depths at its keypoints)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    embed = torch.randn((width, 3 * PATCH * PATCH), generator=gen, device=device).bfloat16() / 16
    head = (torch.randn((channels * PATCH * PATCH, width), generator=gen, device=device) / math.sqrt(width)).bfloat16()
    rotary = Rotary(width // heads, axes=2, base=100.0, device=device)
    net = [Layer(width, heads, frames, bits, rotary, gen, device) for _ in range(layers)]
    r = torch.arange(TOKENS, device=device)
    positions = torch.stack((r // COLS, r % COLS), -1).int()
    blocks = torch.arange(frames * FRAME_BLOCKS, dtype=torch.int32, device=device).view(frames, FRAME_BLOCKS)
    scene = torch.randn((3, ROWS * PATCH, COLS * PATCH), generator=gen, device=device)
    summaries, kept, error, depths = [], [], 0.0, None
    for f in range(frames):
        image = torch.roll(scene, 8 * f, 2) + 0.1 * torch.randn(scene.shape, generator=gen, device=device)
        patches = image.view(3, ROWS, PATCH, COLS, PATCH).permute(1, 3, 0, 2, 4).reshape(TOKENS, -1).bfloat16()
        x = patches @ embed.t()
        # the kept frames that are most like this one, by their mean tokens
        mean = torch.nn.functional.normalize(x.float().mean(0), dim=0)
        chosen = []
        if summaries:
            chosen = torch.topk(torch.stack(summaries) @ mean, min(like, f)).indices.tolist()
        seen = torch.cat([blocks[i] for i in chosen] + [blocks[f]])[None]
        lengths = torch.full((1,), seen.shape[1] * BLOCK, dtype=torch.int32, device=device)
        for i, layer in enumerate(net):
            x, (q, k, v, o) = layer(x, positions, blocks[f:f + 1], seen, lengths)
            if i == 0:
                kept.append((k, v))
                if f == frames - 1:
                    want = plain_attention(q, torch.cat([kept[j][0] for j in chosen + [f]]),
                                           torch.cat([kept[j][1] for j in chosen + [f]]))
                    error = float((o.float() - want).norm() / want.norm())
        summaries.append(mean)
        maps = (x @ head.t()).view(ROWS, COLS, PATCH, PATCH, channels).permute(0, 2, 1, 3, 4).float()
        maps = maps.reshape(1, ROWS * PATCH, COLS * PATCH, channels)
        pix = torch.rand((1000, 2), generator=gen, device=device) * torch.tensor([COLS * PATCH, ROWS * PATCH], device=device)
        depths = sample_depth_maps(maps, torch.tensor([len(pix)], device=device), pix, insert_ones=True)
    return error, depths, net


def main():
    p = argparse.ArgumentParser(description=__doc__.split('\n')[0])
    p.add_argument('--frames', type=int, default=8)
    p.add_argument('--layers', type=int, default=2)
    p.add_argument('--bits', choices=['fp8', 'int8'], default='fp8')
    a = p.parse_args()
    bits = torch.float8_e4m3fn if a.bits == 'fp8' else torch.int8
    error, depths, net = run(a.frames, a.layers, bits=bits)
    size = sum(t.numel() * t.element_size() for n in net for t in (n.cache.k, n.cache.v, n.cache.scales))
    print(f'{a.frames} frames kept in {size / 2 ** 20:.1f} MiB ({a.bits}), attention off by {error:.2%}, '
          f'{depths.shape[0]} keypoints x {depths.shape[1]} depth channels')


if __name__ == '__main__':
    main()
