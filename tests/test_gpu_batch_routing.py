"""Router statistics of a ragged batch (GptOssModel.forward_batch): they count the tokens that sequences have, and no padding,
whatever that holds."""
from __future__ import annotations

import pytest
import torch

from nurostream_amd.model.batch import BatchKV

pytestmark = pytest.mark.gpu

TAILS = [[12, 30, 31], [8], [77, 9], [30, 12, 4, 4, 4], []]


def _load(tmp_path, resident):
    from api_cases import write_gptoss_gguf
    from nurostream_amd import synth
    from nurostream_amd.api import NeuroStream
    from nurostream_amd.format.gguf import GGMLType
    cfg = synth.MoEConfig("s", GGMLType.MXFP4, 8, 4, 256, 192, "gptoss", "clamped_swiglu", True, torch.bfloat16)
    path = tmp_path / "tiny.gguf"
    write_gptoss_gguf(path, cfg, n_layers=2, seed=4, attention=True)
    kw = dict(slab_budget="1GB") if resident else dict(mem_budget="64MB")
    ns = NeuroStream.load(path, device="cuda", vram_budget="1GB", block_rows=64, **kw)
    assert all((ns.model._fused_layer(li) is not None) == resident for li in range(2))
    return ns, cfg


def _ragged(ns, dev, padding, counts=True):
    """Two steps of a ragged batch -> (the statistics that they add, logits of the sequences that have tokens)."""
    from nurostream_amd.moe.router import RouterStats
    model = ns.model
    model.router_stats = RouterStats()
    kv = BatchKV(ns.cfg.n_layer, model.attn_config(), len(TAILS), 6, dev)
    ids = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    out = []
    for cut in ([t[:3] for t in TAILS], [t[3:] for t in TAILS]):
        n = max(map(len, cut))
        got = model.forward_batch(ids([c + [padding] * (n - len(c)) for c in cut]), kv, ids([len(c) for c in cut]) if counts else None)
        out += [got[b] for b, c in enumerate(cut) if c]
    return model.router_stats, out


@pytest.mark.parametrize("resident", [True, False], ids=["resident", "streamed"])
def test_padding_is_not_counted(dev, tmp_path, resident):
    ns, cfg = _load(tmp_path, resident)
    live = sum(map(len, TAILS))
    runs = [_ragged(ns, dev, padding) for padding in (0, 250)]
    for st, _ in runs:
        assert st.tokens_routed == 2 * live
        assert sum(st.hits.values()) == 2 * live * cfg.top_k and min(st.hits.values()) > 0
    assert runs[0][0].hits == runs[1][0].hits
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))
    st, _ = _ragged(ns, dev, 0, counts=False)  # without counts all tokens are in earnest
    assert st.tokens_routed == 2 * 5 * (3 + 2) and sum(st.hits.values()) == 2 * 25 * cfg.top_k


@pytest.mark.parametrize("resident", [True, False], ids=["resident", "streamed"])
def test_a_step_of_ended_sequences(dev, tmp_path, resident):
    ns, _ = _load(tmp_path, resident)
    kv = BatchKV(ns.cfg.n_layer, ns.model.attn_config(), 3, 2, dev)
    before = ns.model.router_stats.tokens_routed
    counts = torch.tensor([0, 0, -1], dtype=torch.int32, device=dev)
    got = ns.model.forward_batch(torch.ones(3, 1, dtype=torch.int32, device=dev), kv, counts)
    assert got.shape[0] == 3 and kv.pos.tolist() == [0, 0, 0]
    assert ns.model.router_stats.tokens_routed == before and not ns.model.router_stats.hits


def test_generate_batch_counts_what_it_runs(dev, tmp_path):
    """Prompts of different lengths and an answer that ends early: every token once per layer, the last drawn ones aside."""
    ns, cfg = _load(tmp_path, True)
    prompts = [[5, 6, 7, 9, 1, 2], [5, 6], [5, 6, 8]]
    steps = list(ns.generate_batch(prompts, max_tokens=4, stop_on_eos=False))
    st = ns.model.router_stats
    # (the first token is shared: run once; then 5, 1 and 2 of the prompts, and three of the four drawn of each)
    assert len(steps) == 4 and st.tokens_routed == 2 * (1 + 5 + 1 + 2 + 3 * 3)
    assert sum(st.hits.values()) == st.tokens_routed * cfg.top_k


def test_a_captured_pass_of_ragged_steps(dev, tmp_path):
    """A pass captured as the model's own decode graph is (no statistics on the way) serves other tokens and counts."""
    ns, _ = _load(tmp_path, True)
    model, c = ns.model, ns.model.attn_config()
    eager, kept = (BatchKV(ns.cfg.n_layer, c, 3, 8, dev) for _ in "ab")
    tokens, counts = torch.ones(3, 2, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    model.forward_batch(tokens, kept, counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    model._capturing = []
    try:
        with torch.cuda.graph(graph):
            logits = model.forward_batch(tokens, kept, counts)
    finally:
        model._capturing = None
    kept.reset()
    for step in range(4):
        fresh = torch.tensor([[5 + step, 9], [40, 7 * step], [3, 200 + step]], dtype=torch.int32, device=dev)
        some = torch.tensor([1 + step % 2, 2 - step % 2, int(step < 2)], dtype=torch.int32, device=dev)
        want = model.forward_batch(fresh, eager, some)
        tokens.copy_(fresh)
        counts.copy_(some)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want) and torch.equal(kept.pos, eager.pos), step
