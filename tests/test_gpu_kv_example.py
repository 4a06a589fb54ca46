"""The paged-cache example: a pruned layer with its cache, against its definitions."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("paged_decode", os.path.join(ROOT, "examples", "paged_decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def dense(csr, rows, cols):
    ip, ix, v = csr
    d = torch.zeros(rows, cols, dtype=torch.float64)
    d[torch.repeat_interleave(torch.arange(rows), torch.from_numpy(np.diff(ip))), torch.from_numpy(ix)] = torch.from_numpy(v).double()
    return d


@pytest.mark.parametrize("cache,prefix,prompts", [("bf16", 200, (5, 33, 0, 64)), ("f16", 0, (7, 1, 40)), ("f32", 33, (0, 0, 3))])
def test_serving_a_pruned_layer(cache, prefix, prompts):
    seen = []

    def each(layer, batch, qkv, a, y):
        torch.cuda.synchronize()
        H, K, D, page = layer.heads, layer.kv_heads, layer.dim, batch.page
        T = qkv.shape[0]
        start, lengths = batch.start.cpu().numpy(), batch.lengths.cpu().numpy()
        table, kp, vp = batch.table.cpu().numpy(), layer.k_pool.cpu(), layer.v_pool.cpu()
        host = qkv.cpu()
        k, v = (host[:, (H + i * K) * D:(H + (i + 1) * K) * D].reshape(T, K, D).to(kp.dtype) for i in range(2))
        # every new token's key and value stand where its request's table says
        for b in range(batch.B):
            for i in range(start[b + 1] - start[b]):
                key = lengths[b] - (start[b + 1] - start[b]) + i
                p = table[b, key // page]
                assert torch.equal(kp[p, :, key % page], k[start[b] + i]) and torch.equal(vp[p, :, key % page], v[start[b] + i])
        want, bound = R.attention(host[:, :H * D].reshape(T, H, D), kp, vp, D ** -0.5, batch.prefix_table.cpu().numpy(),
                                  batch.prefix_len, table, lengths, start, "f32")
        assert bool(((a.cpu().double().reshape(T, H, D) - want).abs() <= bound).all())
        # fast products: within 1e-5 of the 64-bit ones, normwise
        ref = a.cpu().double() @ dense(layer.o_host, layer.hidden, H * D).T
        assert float((y.cpu().double() - ref).norm()) <= 1e-5 * float(ref.norm()) + 1e-30
        seen.append(T)

    b = example().serve(prefix=prefix, prompts=prompts, steps=3, cache=cache, each=each)
    assert seen == [sum(prompts)] + [len(prompts)] * 3
    assert b.lengths.tolist() == [n + 3 for n in prompts]
