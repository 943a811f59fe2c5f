"""A decoder layer that answers from a cache of bounded size.

Up to eight sequences go through one layer: attention over a paged cache, then
the sparse MLP. Their prompts come in chunks of different lengths (one call
takes a chunk of each), the softmax weight that every cached slot receives is
summed on the way, and once a cache has grown by `slack` tokens past `budget`
it is cut back to its heaviest slots: into a second set of pages, the sets
taking turns. Decoding is one token of each sequence per step.

    python examples/bounded_cache.py [--sequences 4] [--prompt 6000] [--steps 256]

Weights and inputs are random; torch does the projections and the norm before
the attention.
"""
import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from leanstream_b200 import PagedAttention, evict_cache  # noqa: E402
from leanstream_b200.batch import BatchMLP, union_plan  # noqa: E402
from leanstream_b200.synthetic import make_layer  # noqa: E402


class BoundedLayer:
    def __init__(self, sequences, longest, *, hidden=1024, q_heads=16, kv_heads=4, head_dim=64, page=16, budget=512,
                 slack=64, sinks=4, recent=64, chunk=512, groups=16, seed=0, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        half, int32 = dict(dtype=torch.float16, device=device), dict(dtype=torch.int32, device=device)
        self.sequences, self.hidden, self.page, self.chunk = sequences, hidden, page, chunk
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.budget, self.slack, self.sinks, self.recent = budget, slack, sinks, recent
        rows = (q_heads + 2 * kv_heads) * head_dim
        self.w_qkv = torch.randn(hidden, rows, generator=gen, device=device).mul_(hidden ** -0.5).half()
        self.w_out = torch.randn(q_heads * head_dim, hidden, generator=gen, device=device).mul_(hidden ** -0.5).half()

        # pages: the prompt's, then two sets for what is kept and the tokens after it
        long, short = -(-longest // page), -(-(budget + slack) // page)
        pool = sequences * (long + 2 * short)
        self.k_pages, self.v_pages = (torch.zeros(pool, page, kv_heads, head_dim, **half) for _ in range(2))
        order = torch.randperm(pool, generator=gen, device=device).int()
        self.tables = [o.reshape(sequences, -1) for o in order.split([sequences * n for n in (long, short, short)])]
        self.table, self.turn = self.tables[0], 0
        self.kv_len = torch.zeros(sequences, **int32)
        self.lengths = [0] * sequences  # the same on the host: they follow from the calls
        self.weights = torch.zeros(sequences, kv_heads, max(long, short) * page, device=device)
        self.kept = torch.empty(sequences, kv_heads, budget, **int32)
        self.kept_weights = torch.empty(sequences, kv_heads, budget, device=device)
        self.error = torch.zeros(1, **int32)
        self.attention = PagedAttention(q_heads, kv_heads, head_dim, page_size=page, max_sequences=sequences,
                                        max_tokens=sequences * chunk, max_queries=chunk,
                                        max_weights_length=self.weights.shape[2], device=device)
        self.one_each = torch.arange(sequences + 1, **int32)

        layer = make_layer(seed, hidden, groups)
        _, descs, mask = union_plan([[(b + i) % groups for i in range(groups // 2)] for b in range(sequences)])
        self.mlp = BatchMLP(hidden, 64, groups, device=device)
        self.mlp_args = dict(
            cache=torch.from_numpy(layer.packed).to(device), union_count=len(descs),
            scales=torch.from_numpy(layer.scales.reshape(-1).view("int16")).view(torch.float16).to(device),
            union_descs=torch.from_numpy(descs.reshape(-1).view("int32").copy()).to(device),
            mask=torch.from_numpy(mask.copy()).to(device), norm_input=True)

    def attend(self, x, q_start, counts):
        """x [tokens][hidden], counts[b] of them of sequence b: x + attention."""
        qkv = (torch.nn.functional.rms_norm(x, (self.hidden,)) @ self.w_qkv).view(len(x), -1, self.head_dim)
        q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], dim=1)
        out = torch.empty(len(x), self.q_heads, self.head_dim, dtype=x.dtype, device=x.device)
        self.lengths = [n + c for n, c in zip(self.lengths, counts)]
        self.kv_len += q_start.diff()
        self.attention.run(q=q, output=out, k_pages=self.k_pages, v_pages=self.v_pages, page_table=self.table,
                           q_start=q_start, kv_len=self.kv_len, max_q=max(counts), k_new=k, v_new=v,
                           weights=self.weights[:, :, :self.table.shape[1] * self.page])
        return x + out.flatten(1) @ self.w_out

    def evict(self):
        """Cuts every sequence to the budget, in the pages whose turn it is."""
        self.turn = 1 if self.turn != 1 else 2
        new, new_len = self.tables[self.turn], torch.empty_like(self.kv_len)
        evict_cache(k_pages=self.k_pages, v_pages=self.v_pages, page_table=self.table, kv_len=self.kv_len,
                    weights=self.weights[:, :, :self.table.shape[1] * self.page], budget=self.budget, new_table=new,
                    new_len=new_len, kept=self.kept, sinks=self.sinks, recent=self.recent,
                    new_weights=self.kept_weights, error=self.error)
        self.table, self.kv_len = new, new_len
        self.weights[:, :, :self.budget] = self.kept_weights
        self.lengths = [min(n, self.budget) for n in self.lengths]

    def feed_forward(self, x):
        y, out = torch.empty_like(x), torch.empty_like(x)
        self.mlp.run(x=x, output=y, residual=x, hidden_out=out, tokens=len(x), **self.mlp_args)
        return out

    def prompt(self, xs):
        """xs[b] [tokens][hidden]: the layer's output at each last token."""
        last = [None] * self.sequences
        for at in range(0, max(len(x) for x in xs), self.chunk):
            parts = [x[at:at + self.chunk] for x in xs]
            counts = [len(x) for x in parts]
            starts = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(self.kv_len.device)
            done = self.attend(torch.cat(parts), starts, counts).split(counts)
            last = [d[-1] if len(d) else l for d, l in zip(done, last)]
        self.evict()
        return self.feed_forward(torch.stack(last))

    def step(self, x):
        """One token of each sequence, x [sequences][hidden]."""
        if max(self.lengths) >= self.budget + self.slack:
            self.evict()
        return self.feed_forward(self.attend(x, self.one_each, [1] * self.sequences))

    def check(self):
        """Raises when a call reported bad lengths or pages, or gave up a wait."""
        found = self.attention.error() | int(self.error.item()) | self.mlp.error()
        if found:
            raise RuntimeError(f"error bits {found:#x}")


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--sequences", type=int, default=4)
    parser.add_argument("--prompt", type=int, default=6000, help="tokens of the longest prompt")
    parser.add_argument("--steps", type=int, default=256)
    args = parser.parse_args()
    layer = BoundedLayer(args.sequences, args.prompt)
    lengths = [max(1, args.prompt * (b + 1) // args.sequences) for b in range(args.sequences)]
    xs = [torch.randn(n, layer.hidden, device="cuda").half() for n in lengths]
    layer.prompt(xs)
    layer = BoundedLayer(args.sequences, args.prompt)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    x = layer.prompt(xs)
    torch.cuda.synchronize()
    middle = time.perf_counter()
    for _ in range(args.steps):
        x = layer.step(torch.nn.functional.rms_norm(x, (layer.hidden,)))
    torch.cuda.synchronize()
    end = time.perf_counter()
    layer.check()
    print(f"prompts of {lengths} tokens: {1e3 * (middle - begin):.2f} ms; cut to {layer.budget} slots; "
          f"{args.steps} steps of {args.sequences} tokens: {1e6 * (end - middle) / max(1, args.steps):.0f} us each")


if __name__ == "__main__":
    main()
