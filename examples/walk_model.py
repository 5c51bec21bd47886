"""A sequence model over temporal walks, trained and served with the operators.

    python examples/walk_model.py [--walks 4096] [--length 80] [--steps 50]

1. The engine samples walks from a graph of events whose nodes meet within
   groups; the model learns to name a walk's next node.
2. Training: each layer's attention is ``walk_attention`` over the walks as the
   sampler pads them, with a learned bias by distance and a decay by time.
3. Serving: the caches are filled from the first events of some walks, then
   ``walk_attention_step`` takes one event of each walk at a time; the logits are
   compared with those of one pass over whole walks.
4. A look inside: ``relative_bias`` gives the learned bias as a dense array, from
   which plain tensor code shows how far back each head looks.
"""
import argparse
import math
import os
import sys
import time

import torch  # before the engine: its HIP runtime has to come up first
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..",
                                "temporal-random-walk_amd"))
from temporal_random_walk import TemporalRandomWalk  # noqa: E402
from temporal_random_walk import operators as ops  # noqa: E402

HEADS, KV_HEADS, DIM = 8, 2, 64
WIDTH = HEADS * DIM
BUCKETS, REACH = 32, 128


def sample_walks(nodes, group, walks, length, seed):
    """Nodes [walks, length], times in units of the whole span, lengths; on the GPU."""
    gen = torch.Generator().manual_seed(seed)
    events = 100 * nodes
    source = torch.randint(nodes, (events,), generator=gen)
    target = source // group * group + torch.randint(group, (events,), generator=gen)
    when = torch.arange(events)
    graph = TemporalRandomWalk(is_directed=False, use_gpu=True, global_seed=seed + 1)
    graph.add_multiple_edges(source.int().numpy(), target.int().numpy(), when.numpy())
    at, t, lens = graph.get_random_walks_and_times_for_all_nodes(
        max_walk_len=length, walk_bias="ExponentialIndex", num_walks_per_node=-(-walks // nodes))[:3]
    at, t, lens = (torch.as_tensor(x[:walks].astype("int64")).cuda() for x in (at, t, lens))
    seen = torch.arange(length, device="cuda") < lens[:, None]
    return at.where(seen, 0), (t.float() / events).where(seen, 0), lens


class Layer(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm, self.norm_mlp = nn.LayerNorm(WIDTH), nn.LayerNorm(WIDTH)
        self.qkv = nn.Linear(WIDTH, (HEADS + 2 * KV_HEADS) * DIM)
        self.out = nn.Linear(WIDTH, WIDTH)
        self.mlp = nn.Sequential(nn.Linear(WIDTH, 4 * WIDTH), nn.GELU(),
                                 nn.Linear(4 * WIDTH, WIDTH))

    def project(self, x):
        """q, k and v: views of one projection, as the operators take them."""
        qkv = self.qkv(self.norm(x)).unflatten(-1, (HEADS + 2 * KV_HEADS, DIM))
        return qkv.split([HEADS, KV_HEADS, KV_HEADS], dim=-2)

    def rest(self, x, attention):
        x = x + self.out(attention.flatten(-2))
        return x + self.mlp(self.norm_mlp(x))


class WalkModel(nn.Module):
    def __init__(self, nodes, layers=2):
        super().__init__()
        self.embed = nn.Embedding(nodes, WIDTH)
        self.layers = nn.ModuleList(Layer() for _ in range(layers))
        self.bias = nn.Parameter(torch.zeros(HEADS, BUCKETS))
        self.norm, self.head = nn.LayerNorm(WIDTH), nn.Linear(WIDTH, nodes)
        self.register_buffer("buckets", ops.distance_buckets(BUCKETS, REACH, device="cpu"))
        self.register_buffer("slopes", 2.0 ** -torch.arange(HEADS).float())

    def terms(self):
        return dict(bias_table=self.bias, buckets=self.buckets, slopes=self.slopes)

    def forward(self, at, times, mask, caches=None):
        """Logits at each event of padded walks; fills the caches' first positions if given."""
        x = self.embed(at)
        for i, layer in enumerate(self.layers):
            q, k, v = layer.project(x)
            if caches:
                for cache, rows in zip(caches[i], (k, v)):
                    cache[:, :rows.shape[1]] = rows
            x = layer.rest(x, ops.walk_attention(q, k, v, mask, times=times, **self.terms()))
        return self.head(self.norm(x))

    def step(self, at, times, caches, k_times, lens):
        """Logits after one new event of each walk."""
        x = self.embed(at)
        for layer, (k_cache, v_cache) in zip(self.layers, caches):
            q, k, v = layer.project(x)
            x = layer.rest(x, ops.walk_attention_step(
                q, k, v, k_cache, v_cache, lens, times=times, k_times=k_times, **self.terms()))
        return self.head(self.norm(x))


def train(model, at, times, lens, steps, batch):
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    length, losses = at.shape[1], []
    target_at = torch.arange(1, length, device="cuda")
    for n in range(steps):
        pick = torch.arange(n * batch, (n + 1) * batch, device="cuda") % at.shape[0]
        a, t, m = at[pick], times[pick], lens[pick]
        mask = ops.WalkMask.padded(m, length)  # once for all layers and both directions
        with torch.autocast("cuda", torch.bfloat16):
            logits = model(a, t, mask)[:, :-1]
        target = a[:, 1:].where(target_at < m[:, None], -100)
        loss = F.cross_entropy(logits.flatten(0, 1).float(), target.flatten(), ignore_index=-100)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def serve(model, at, times, lens, prompt):
    """One event of each walk at a time after a prompt: how many events, and how far their logits
    are from one pass's."""
    batch, length = at.shape
    with torch.autocast("cuda", torch.bfloat16):
        whole = model(at, times, ops.WalkMask.padded(lens, length)).float()
        caches = [tuple(torch.zeros(batch, length, KV_HEADS, DIM, dtype=torch.bfloat16,
                                    device="cuda") for _ in "kv") for _ in model.layers]
        k_times = torch.zeros(batch, length, device="cuda")
        k_times[:, :prompt] = times[:, :prompt]
        held = lens.clamp(max=prompt)
        model(at[:, :prompt], times[:, :prompt].contiguous(), ops.WalkMask.padded(held, prompt),
              caches)
        off, size = [], []
        for n in range(prompt, length):
            here = n < lens
            now = torch.where(here, held, -1)  # walks that have ended are idle
            logits = model.step(at[:, n], times[:, n].contiguous(), caches, k_times, now).float()
            held = held + here
            off.append((logits - whole[:, n])[here].square().sum())
            size.append(whole[:, n][here].square().sum())
    served = int((lens - prompt).clamp(min=0).sum())
    return served, float(torch.stack(off).sum() / torch.stack(size).sum().clamp(min=1e-30)) ** 0.5


@torch.no_grad()
def look(model, at, times, lens):
    """How many events back each head of the first layer looks, on average."""
    length = at.shape[1]
    q, k, _ = (x.float().transpose(1, 2) for x in model.layers[0].project(model.embed(at)))
    scores = q @ k.repeat_interleave(HEADS // KV_HEADS, 1).mT.contiguous() / math.sqrt(DIM)
    scores += ops.relative_bias(model.bias, model.buckets, length, length)
    scores -= model.slopes[:, None, None] * (times[:, None, :, None] - times[:, None, None]).abs()
    place = torch.arange(length, device="cuda")
    back = place[:, None] - place
    share = scores.masked_fill(back < 0, -math.inf).softmax(-1)
    mean = (share * back).sum(-1)
    real = (place < lens[:, None])[:, None].expand_as(mean)
    return (mean * real).sum((0, 2)) / real.sum((0, 2))


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--nodes", type=int, default=4000)
    parser.add_argument("--walks", type=int, default=8000)
    parser.add_argument("--length", type=int, default=80)
    parser.add_argument("--batch", type=int, default=1000)
    parser.add_argument("--steps", type=int, default=50)
    args = parser.parse_args(argv)
    torch.manual_seed(0)
    at, times, lens = sample_walks(args.nodes, 20, args.walks, args.length, seed=0)
    print(f"{at.shape[0]} walks, {int(lens.sum())} events")
    model = WalkModel(args.nodes).cuda()
    torch.cuda.synchronize()
    began = time.perf_counter()
    losses = train(model, at, times, lens, args.steps, args.batch)
    took = time.perf_counter() - began
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {args.steps} steps, "
          f"{args.steps / took:.1f} steps/s")
    some = torch.arange(min(256, at.shape[0]), device="cuda")
    prompt = args.length // 2
    served, off = serve(model, at[some], times[some], lens[some], prompt)
    print(f"{served} events served from event {prompt} on: logits {off:.2e} from those of one pass")
    far = look(model, at[some], times[some], lens[some])
    print("events that a head looks back:", " ".join(f"{x:.1f}" for x in far.tolist()))
    return losses, served, off, far


if __name__ == "__main__":
    main()
