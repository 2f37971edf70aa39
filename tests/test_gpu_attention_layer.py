"""The example layer: quantised projections, append and attention together, as prompts, in chunks and as a replayed decode step."""
import numpy as np
import pytest
import torch

import avelang_amd as ave
from examples.attention_layer import AttentionLayer, main
from tests import attention_helpers as A

pytestmark = pytest.mark.gpu


def _layer(gpu, head_dim=64):
    return AttentionLayer(512, 8, 2, head_dim, 3, 120, 16, device=gpu)


def _reference(layer, lengths, before):
    """Attention in fp64 over what the cache holds, for the queries that the layer made; and a bound."""
    batch = A.Batch.__new__(A.Batch)
    batch.rows = [(n, n + b) for n, b in zip(lengths, before)]
    batch.hq, batch.hkv, batch.d = layer.heads, layer.kv_heads, layer.head_dim
    batch.cu = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    batch.q = layer.q.float().cpu().numpy()
    batch.k, batch.v = [], []
    for b, (_, keys) in enumerate(batch.rows):
        at = torch.arange(keys, device=layer.q.device)
        slots = (layer.page_table[b][at // layer.page_size] * layer.page_size + at % layer.page_size).int()
        for x, into in zip(ave.gather_kv_mxfp4(layer.cache, slots), (batch.k, batch.v)):
            into.append(x.double().cpu().numpy())
    out, _, tol, _ = batch.reference()
    return out, tol


@pytest.mark.parametrize("head_dim", [64, 128])
def test_prompts_and_chunks_against_fp64(gpu, head_dim):
    layer = _layer(gpu, head_dim)
    g = torch.Generator().manual_seed(1)
    before = [0, 0, 0]
    for lengths in ([40, 1, 17], [3, 50, 1], [1, 1, 1]):
        x = torch.randn(sum(lengths), 512, generator=g).bfloat16().to(gpu)
        y, seq_lens = layer.prompts(x, lengths, before)
        want, tol = _reference(layer, lengths, before)
        assert (np.abs(layer.attended.float().cpu().numpy() - want) <= tol).all()
        again = ave.gemm_mxfp4_transposed_b(*ave.quantize_mxfp4(layer.attended.view(len(x), -1)), *layer.out)
        assert torch.equal(y, again) and y.isfinite().all()
        before = [b + n for b, n in zip(before, lengths)]
        assert seq_lens.tolist() == before


def test_replayed_decode_steps_equal_eager_ones(gpu):
    layer, eager = _layer(gpu), _layer(gpu)
    lengths = [30, 64, 5]
    x = torch.randn(sum(lengths), 512, generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    _, lens = layer.prompts(x, lengths)
    eager.prompts(x, lengths)
    steps = torch.randn(6, 3, 512, generator=torch.Generator().manual_seed(3)).bfloat16().to(gpu)
    x, now = steps[0].clone(), lens + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, now)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, now)
    for i in range(6):
        x.copy_(steps[i])
        now.copy_(lens + 1 + i)
        graph.replay()
        want = eager(steps[i], lens + 1 + i)
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
    assert all(torch.equal(a, b) for a, b in zip(layer.cache, eager.cache))


def test_the_example_runs(gpu, capsys):
    main(hidden=512, heads=8, kv_heads=2, head_dim=64, lengths=(50, 3), steps=4)
    said = capsys.readouterr().out
    assert said.count("finite True") == 2
