"""The attention half of a decoder layer with everything large in MXFP4: weights, the key/value cache, and the activations that go
into the matrix products.

    x -> quantize -> qkv projection -> norm + rotation + append -> attention over the cache -> quantize -> output projection

Prompts of different lengths go in side by side, whole or in chunks; then a decode step is captured once in a graph and replayed.
Run it: ``python examples/attention_layer.py``."""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import avelang_amd as ave  # noqa: E402


class AttentionLayer:
    """Weights of one layer and its cache for ``sequences`` of at most ``max_len`` tokens; random ones, for the want of others."""

    def __init__(self, hidden, heads, kv_heads, head_dim, sequences, max_len, page_size=64, *, device="cuda", seed=0):
        self.heads, self.kv_heads, self.head_dim, self.page_size = heads, kv_heads, head_dim, page_size
        g = torch.Generator().manual_seed(seed)
        weight = lambda n, k: ave.quantize_mxfp4((torch.randn(n, k, generator=g) * k ** -0.5).to(device))   # noqa: E731
        self.qkv, self.out = weight((heads + 2 * kv_heads) * head_dim, hidden), weight(hidden, heads * head_dim)
        self.q_weight, self.k_weight = (torch.ones(head_dim, dtype=torch.bfloat16, device=device) for _ in range(2))
        angle = torch.arange(max_len)[:, None] * 10000.0 ** (-torch.arange(0, head_dim, 2) / head_dim)
        self.cos, self.sin = angle.cos().to(device), angle.sin().to(device)
        per_sequence = -(-max_len // page_size)
        self.cache = ave.kv_cache_mxfp4(sequences * per_sequence, kv_heads, page_size, head_dim, device)
        self.page_table = torch.randperm(sequences * per_sequence, generator=g).int().view(sequences, per_sequence).to(device)

    def __call__(self, x, seq_lens, cu_q=None, sequence_of=None, max_q=1):
        """``x`` bf16 ``[T, hidden]``: the last ``cu_q[b+1] - cu_q[b]`` tokens of sequence ``b`` (``cu_q`` ``None``: one token each), which is
        ``seq_lens[b]`` long with them; ``sequence_of`` int64 ``[T]``: the sequence of each row.  All on the device, nothing is read back."""
        t = x.shape[0]
        if cu_q is None:
            positions, row = seq_lens - 1, slice(None)
        else:
            row = sequence_of
            positions = (torch.arange(t, device=x.device) - cu_q[1:][row] + seq_lens[row]).int()
        page = self.page_table[row].gather(1, (positions // self.page_size).long()[:, None])[:, 0]
        slots = page * self.page_size + positions % self.page_size
        qkv = ave.gemm_mxfp4_transposed_b(*ave.quantize_mxfp4(x), *self.qkv).view(t, -1, self.head_dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
        q = ave.append_kv_mxfp4(k, v, self.cache, slots, self.cos, self.sin, positions, self.k_weight, q=q, q_weight=self.q_weight)
        self.q = q      # (kept for whoever wants to look)
        self.attended = ave.attention_mxfp4(q, self.cache, self.page_table, seq_lens, cu_q, max_q=max_q)
        return ave.gemm_mxfp4_transposed_b(*ave.quantize_mxfp4(self.attended.view(t, -1)), *self.out)

    def prompts(self, x, lengths, before=None):
        """Rows of several sequences one after the other, ``lengths[b]`` each (a list), behind ``before[b]`` tokens that are there already."""
        new = torch.tensor(lengths, dtype=torch.int32)
        cu_q = torch.cat([torch.zeros(1, dtype=torch.int32), new.cumsum(0).int()]).to(x.device)
        sequence_of = torch.repeat_interleave(torch.arange(len(lengths)), new.long()).to(x.device)
        seq_lens = (new + torch.tensor(before or [0] * len(lengths), dtype=torch.int32)).to(x.device)
        return self(x, seq_lens, cu_q, sequence_of, max(lengths)), seq_lens


def main(hidden=4096, heads=32, kv_heads=8, head_dim=128, lengths=(1000, 37, 512, 2048), steps=32):
    layer = AttentionLayer(hidden, heads, kv_heads, head_dim, len(lengths), max(lengths) + steps + 1)
    x = torch.randn(sum(lengths), hidden, device="cuda").bfloat16()
    y, seq_lens = layer.prompts(x, list(lengths))
    torch.cuda.synchronize()
    print(f"prompts of {list(lengths)} tokens: out {tuple(y.shape)}, finite {bool(y.isfinite().all())}")

    x = torch.randn(len(lengths), hidden, device="cuda").bfloat16()
    lens = seq_lens + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, lens)                                     # first launches outside the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, lens)
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(steps):
        graph.replay()
        x.copy_(y)
        lens += 1
    torch.cuda.synchronize()
    print(f"{steps} decode steps of {len(lengths)} sequences: {(time.perf_counter() - start) / steps * 1e6:.1f} us each, finite {bool(y.isfinite().all())}")


if __name__ == "__main__":
    main()
