"""Next-patch prediction on point clouds of different sizes, with every operator of the
package in the place where a network uses it.

A cloud is cut into patches: furthest point sampling picks centres, knn the points around
each, and a patch becomes a token.  The clouds' tokens lie packed one after another
(no padding) and pass through pre-norm blocks of layer norm and causal packed
attention; token i predicts the points of patch i + 1, scored by the chamfer distance.
Generation feeds one token at a time: each block keeps its keys and values in a cache
and reads them with cached attention.

    python examples/patch_tokens.py [--steps 60] [--clouds 6] [--dtype bfloat16]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch_point_ops_b200 as tpo  # noqa: E402

WIDTH, HEADS, KV_HEADS, PATCH = 128, 4, 2, 16


class Block(torch.nn.Module):
    """x + attention(norm(x)), then x + mlp(norm(x)); grouped heads."""

    def __init__(self):
        super().__init__()
        self.head = WIDTH // HEADS
        self.norm1, self.norm2 = tpo.LayerNorm(WIDTH), tpo.LayerNorm(WIDTH)
        self.qkv = torch.nn.Linear(WIDTH, (HEADS + 2 * KV_HEADS) * self.head)
        self.out = torch.nn.Linear(WIDTH, WIDTH)
        self.mlp = torch.nn.Sequential(torch.nn.Linear(WIDTH, 2 * WIDTH), torch.nn.GELU(), torch.nn.Linear(2 * WIDTH, WIDTH))
        self.attention = tpo.PackedAttention(causal=True)

    def heads(self, x):
        qkv = self.qkv(self.norm1(x)).view(x.shape[0], HEADS + 2 * KV_HEADS, self.head)
        return qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)  # views: the operators take their strides

    def rest(self, x, attended):
        x = x + self.out(attended.reshape(x.shape))
        return x + self.mlp(self.norm2(x))

    def forward(self, x, offsets):
        return self.rest(x, self.attention(*self.heads(x), offsets))

    def step(self, x, cache, lengths):
        """One new token per cloud at place lengths[n]; the cache is (2, N, P, KV_HEADS, head)."""
        q, k, v = self.heads(x)
        rows = torch.arange(x.shape[0], device=x.device)
        cache[0, rows, lengths], cache[1, rows, lengths] = k, v
        return self.rest(x, tpo.cached_attention(q, cache[0], cache[1], lengths + 1))


class PatchNet(torch.nn.Module):
    def __init__(self, blocks=2):
        super().__init__()
        self.embed = torch.nn.Linear(3 * PATCH + 3, WIDTH)
        self.blocks = torch.nn.ModuleList(Block() for _ in range(blocks))
        self.norm = tpo.LayerNorm(WIDTH)
        self.points = torch.nn.Linear(WIDTH, 3 * PATCH)

    def read_out(self, x):
        return self.points(self.norm(x)).view(-1, PATCH, 3)

    def forward(self, tokens, offsets):
        x = self.embed(tokens)
        for block in self.blocks:
            x = block(x, offsets)
        return self.read_out(x)

    def caches(self, clouds, places, like):
        return [like.new_zeros(2, clouds, places, KV_HEADS, WIDTH // HEADS) for _ in self.blocks]

    def step(self, tokens, caches, lengths):
        x = self.embed(tokens)
        for block, cache in zip(self.blocks, caches):
            x = block.step(x, cache, lengths)
        return self.read_out(x)


def make_clouds(count, seed=0, device="cuda"):
    """Noisy helices of different lengths: (points (N, 3)) each."""
    g = torch.Generator().manual_seed(seed)
    clouds = []
    for i in range(count):
        n = int(torch.randint(300, 1500, (), generator=g))
        t = torch.linspace(0, 4 + i % 3, n)[:, None]
        xyz = torch.cat([t.cos(), t.sin(), t / 3], 1) + 0.02 * torch.randn(n, 3, generator=g)
        clouds.append(xyz.to(device))
    return clouds


def patches(cloud, per=24):
    """(tokens, patch points relative to their centre) in order of the height of the centres."""
    xyz = cloud[None]
    centres = xyz[0, tpo.furthest_point_sampling(xyz, max(2, cloud.shape[0] // per))[0]]
    centres = centres[centres[:, 2].argsort()][None]
    index, _ = tpo.knn_points(centres, xyz, K=PATCH)
    points = (tpo.knn_gather(xyz, index) - centres[:, :, None])[0]
    return torch.cat([points.flatten(1), centres[0]], 1), points


def pack(clouds):
    tokens, points = zip(*(patches(c) for c in clouds))
    lengths = torch.tensor([len(t) for t in tokens], device=clouds[0].device)
    return torch.cat(tokens), torch.cat(points), lengths, tpo.packed_offsets(lengths)


def next_patch_loss(net, tokens, points, offsets, dtype):
    with torch.autocast("cuda", dtype=dtype, enabled=dtype != torch.float32):
        guess = net(tokens, offsets).float()
    last = torch.zeros(len(tokens), dtype=torch.bool, device=tokens.device)
    last[offsets[1:] - 1] = True  # a cloud's last token has no next patch
    here = (~last).nonzero()[:, 0]
    return tpo.chamfer_loss(guess[here], points[here + 1])


@torch.no_grad()
def generate(net, tokens, lengths, offsets):
    """The predictions of `net` over the given tokens, one token per cloud at a time."""
    count, places = len(lengths), int(lengths.max())
    caches = net.caches(count, places, tokens)
    out = tokens.new_zeros(len(tokens), PATCH, 3)
    for place in range(places):
        at = offsets[:-1] + lengths.clamp(max=place + 1) - 1  # clouds that have ended repeat their last token
        guess = net.step(tokens[at], caches, lengths.clamp(max=place + 1) - 1)
        out[at] = guess
    return out


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--clouds", type=int, default=6)
    ap.add_argument("--dtype", choices=("float32", "bfloat16", "float16"), default="bfloat16")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    tokens, points, lengths, offsets = pack(make_clouds(a.clouds))
    net = PatchNet().cuda()
    opt = torch.optim.AdamW(net.parameters(), lr=2e-3)
    losses = []
    for _ in range(a.steps):
        opt.zero_grad()
        loss = next_patch_loss(net, tokens, points, offsets, getattr(torch, a.dtype))
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    with torch.no_grad():
        whole = net(tokens, offsets)
    apart = generate(net, tokens, lengths, offsets)
    off = float((apart - whole).abs().max() / whole.abs().max())
    print(f"{len(lengths)} clouds, {len(tokens)} patches; chamfer loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps; "
          f"token by token against whole clouds: {off:.1e} apart")
    return losses, off


if __name__ == "__main__":
    main()
