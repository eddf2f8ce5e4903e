"""One attention layer served from packed weights and a 4-bit key/value cache.

Every step runs, all on the GPU and without a host copy: the block tables of the step from the
requests' lengths, the stacked q/k/v projection (EXL3), the write of the new keys and values into
the cache, attention over it, and the output projection (EXL3).  A few requests of different prompt
lengths are prefilled in one step and then decode together; one step is recorded in a CUDA graph.

    python examples/kv4_layer.py
"""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import sushi_b200 as sx  # noqa: E402


def random_linear(in_f, outs, n, g):
    """A packed bank of linears that share their input, stacked along the output: random trellis words
    (n halfwords a 16x16 tile) and seeded sign vectors."""
    out_f = sum(outs)
    words = torch.randint(-32768, 32768, (1, in_f // 16, out_f // 16, n), generator=g, device="cuda", dtype=torch.int32)
    sign = lambda *s: torch.randint(0, 2, s, generator=g, device="cuda").half() * 2 - 1
    return sx.Proj(words.to(torch.int16), sign(len(outs), in_f) * in_f ** -0.5, sign(1, out_f))


class Layer:
    def __init__(self, hidden=512, heads=8, kv_heads=2, head_dim=128, pages=64, page_size=16, n=32, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        q, kv = heads * head_dim, kv_heads * head_dim
        self.cols = [0, q, q + kv, q + 2 * kv]
        self.dec = sx.Decode(sx.Codebook.MCG)
        self.qkv = random_linear(hidden, [q, kv, kv], n, g)
        self.o = random_linear(q, [hidden], n, g)
        self.cache = sx.Kv4Cache(pages, kv_heads, head_dim, page_size)
        self.free = torch.randperm(pages, generator=g, device="cuda").int()
        self.free_count = torch.tensor([pages], dtype=torch.int32, device="cuda")

    def step(self, x, ctx_lens, new_lens, table, max_new):
        """x [tokens, hidden]: the new tokens of every request, back to back.  Returns (output rows, the
        step's block tables); the caller carries kv_lens and free_left into the next step."""
        t = sx.block_tables(ctx_lens, new_lens, table, self.free, self.free_count, self.cache.page_size, x.shape[0])
        q, k, v = sx.linear_shared(x, self.qkv, self.cols, self.dec)
        rows = x.shape[0]
        kv = (rows, self.kv_heads, self.head_dim)
        sx.kv4_write(self.cache, k.reshape(kv), v.reshape(kv), t.slots)
        a = sx.kv4_attention(q.reshape(rows, self.heads, self.head_dim), self.cache, table, t.kv_lens, t.cu_q, max_new)
        return sx.linear(a.reshape(rows, -1), self.o, self.dec), t


def main(prompts=(37, 5, 120), decode=8, seed=1):
    layer = Layer()
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    b, hidden = len(prompts), 512
    width = -(-(max(prompts) + decode) // layer.cache.page_size)
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    tokens = torch.randn((sum(prompts) + b * decode, hidden), generator=g, device="cuda").to(torch.bfloat16)

    out, t = layer.step(tokens[:sum(prompts)], i32([0] * b), i32(prompts), table, max(prompts))
    ctx, layer.free_count = t.kv_lens, t.free_left
    outs, ones = [], i32([1] * b)
    for s in range(decode):
        x = tokens[sum(prompts) + s * b:sum(prompts) + (s + 1) * b]
        out, t = layer.step(x, ctx, ones, table, 1)
        ctx, layer.free_count = t.kv_lens, t.free_left
        outs.append(out)

    # The last decode step once more, recorded and replayed: the lengths are tensors, so a server
    # replays one graph for every step of this batch size.
    back, x = ctx - 1, tokens[-b:].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again, _ = layer.step(x, back, ones, table, 1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, outs[-1]), "the recorded step differs"

    # Each request's last row against its whole sequence in one prompt call.
    worst = 0.0
    for r in range(b):
        fresh = Layer()
        first = sum(prompts[:r])
        seq = torch.cat([tokens[first:first + prompts[r]]] + [tokens[sum(prompts) + s * b + r][None] for s in range(decode)])
        whole, _ = fresh.step(seq, i32([0]), i32([len(seq)]), torch.full((1, width), -1, dtype=torch.int32, device="cuda"), len(seq))
        worst = max(worst, ((whole[-1] - outs[-1][r]).float().norm() / whole[-1].float().norm()).item())
    return worst


if __name__ == "__main__":
    err = main()
    print(f"decode steps against whole prompts: relative difference {err:.2e}")
    assert err < 2e-2
