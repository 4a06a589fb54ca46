"""One pruned attention layer serving a batch behind a shared prefix.

The q, k and v projections are pruned weights stacked into one CSR product;
its rows go to a paged key/value cache, every request attends to a prefix that
the cache holds once and to its own tokens, and a pruned output projection
follows.  Block tables and slots are made on the GPU from the requests'
lengths, so that a step needs nothing from the host but the number of tokens.

    python examples/paged_decode.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from pyflamert_amd import rocm, workloads  # noqa: E402


class Layer:
    """Pruned projections and the paged cache of one layer."""

    def __init__(self, ctx, hidden, heads, kv_heads, dim, page, pages, density=0.3, cache="bf16", seed=0):
        self.ctx, self.hidden, self.heads, self.kv_heads, self.dim = ctx, hidden, heads, kv_heads, dim
        q, k, v, o = (workloads.csr_uniform(m, n, density, 0.05, seed + i) for i, (m, n) in enumerate(
            [(heads * dim, hidden), (kv_heads * dim, hidden), (kv_heads * dim, hidden), (hidden, heads * dim)]))
        self.row = (heads + 2 * kv_heads) * dim
        self.qkv_host, self.o_host = workloads.csr_vstack([q, k, v]), o
        self.wqkv = ctx.csr_upload(self.row, hidden, *self.qkv_host)
        self.wo = ctx.csr_upload(hidden, heads * dim, *o)
        kind = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[cache]
        self.k_pool, self.v_pool = (torch.zeros(pages, kv_heads, page, dim, dtype=kind, device="cuda") for _ in range(2))
        self.cache = ctx.kv_bind(self.k_pool.data_ptr(), self.v_pool.data_ptr(), cache, pages, page, kv_heads, dim)

    def project(self, x):
        """[tokens, (heads + 2 kv heads) * dim] of x [tokens, hidden]."""
        y = torch.empty(x.shape[0], self.row, device="cuda")
        self.ctx.gemm_csr_dev(x.data_ptr(), x.shape[0], self.hidden, self.wqkv, y.data_ptr(), mode="fast")
        return y

    def keep(self, qkv, slots):
        """The keys and values of qkv's rows into their slots."""
        at = qkv.data_ptr() + 4 * self.heads * self.dim
        self.cache.write_dev(at, at + 4 * self.kv_heads * self.dim, qkv.shape[0], slots.data_ptr(), "f32",
                             ldk=self.row, ldv=self.row)

    def attend(self, qkv, batch, max_added):
        out = torch.empty(qkv.shape[0], self.heads * self.dim, device="cuda")
        self.cache.attention_dev(qkv.data_ptr(), qkv.shape[0], self.heads, out.data_ptr(), "f32", ldq=self.row,
                                 prefix_table_ptr=batch.prefix_table.data_ptr(), prefix_len=batch.prefix_len,
                                 table_ptr=batch.table.data_ptr(), table_w=batch.table.shape[1], B=batch.B,
                                 lengths_ptr=batch.lengths.data_ptr(), start_ptr=batch.start.data_ptr(),
                                 max_added=max_added, max_length=batch.table.shape[1] * batch.page)
        return out

    def output(self, a):
        y = torch.empty(a.shape[0], self.hidden, device="cuda")
        self.ctx.gemm_csr_dev(a.data_ptr(), a.shape[0], self.heads * self.dim, self.wo, y.data_ptr(), mode="fast")
        return y


class Batch:
    """Requests behind one prefix: block tables, lengths, the free list."""

    def __init__(self, ctx, B, page, pages, prefix_len, width):
        self.ctx, self.B, self.page, self.prefix_len = ctx, B, page, prefix_len
        n = -(-prefix_len // page)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.prefix_table = torch.arange(max(n, 1), **i32)
        self.free = torch.arange(n, pages, **i32)
        self.table = torch.full((B, width), -1, **i32)
        # lengths and the free list's head go back and forth between two buffers
        self.lengths, self.cached = torch.zeros(B, **i32), torch.zeros(B, **i32)
        self.head, self.next_head, self.status = (torch.zeros(1, **i32) for _ in range(3))
        self.start = torch.zeros(B + 1, **i32)

    def prefix_slots(self):
        return torch.arange(self.prefix_len, device="cuda")  # its pages are 0, 1, ..

    def add(self, added, tokens):
        """Pages and slots for added[b] more tokens of each request, `tokens` in all."""
        self.cached, self.lengths = self.lengths, self.cached
        self.head, self.next_head = self.next_head, self.head
        slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
        self.ctx.kv_tables_dev(self.cached.data_ptr(), added.data_ptr(), self.B, self.page, self.free.data_ptr(),
                               self.free.numel(), self.head.data_ptr(), self.table.data_ptr(), self.table.shape[1],
                               slots.data_ptr(), tokens, self.start.data_ptr(), self.lengths.data_ptr(),
                               self.next_head.data_ptr(), self.status.data_ptr())
        return slots


def step(layer, batch, x, added, max_added):
    """One pass of the layer over the added tokens x; (their projections, their attention, the output)."""
    slots = batch.add(added, x.shape[0])
    qkv = layer.project(x)
    layer.keep(qkv, slots)
    a = layer.attend(qkv, batch, max_added)
    return qkv, a, layer.output(a)


def serve(hidden=512, heads=8, kv_heads=2, dim=64, page=16, prefix=200, prompts=(5, 33, 0, 64), steps=4, cache="bf16",
          seed=0, each=None):
    """Prefix, prompts, then single tokens; each(layer, batch, qkv, attention, output) after every pass."""
    ctx = rocm.Context(0)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    B, longest = len(prompts), max(prompts) + steps
    width = -(-longest // page)
    pages = -(-prefix // page) + B * width
    layer = Layer(ctx, hidden, heads, kv_heads, dim, page, pages, cache=cache, seed=seed)
    batch = Batch(ctx, B, page, pages, prefix, width)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tokens = lambda n: torch.randn(n, hidden, generator=gen, device="cuda")  # noqa: E731
    layer.keep(layer.project(tokens(prefix)), batch.prefix_slots())
    for i in range(1 + steps):
        counts = list(prompts) if i == 0 else [1] * B
        added = torch.tensor(counts, dtype=torch.int32, device="cuda")
        out = step(layer, batch, tokens(sum(counts)), added, max(counts))
        if each is not None:
            each(layer, batch, *out)
    torch.cuda.synchronize()
    if batch.status.item():
        raise RuntimeError("block tables: status %d" % batch.status.item())
    return batch


if __name__ == "__main__":
    b = serve(each=lambda layer, batch, qkv, a, y: print("%d tokens, lengths %s, |y| %.3f" % (
        len(y), batch.lengths.tolist(), y.norm().item())))
    print("pages left: %d" % (b.free.numel() - b.next_head.item()))
