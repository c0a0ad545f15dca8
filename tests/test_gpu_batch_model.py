"""Several sequences at once in the model: forward_batch, generate_batch, and generate's further filters."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from batch_cases import ROWS
from helpers import rel_max, to_np
from nurostream_amd.model.batch import BatchKV, load_rows
from nurostream_amd.model.decode import DeviceKV
from nurostream_amd.model.draft import DraftKV, commit

pytestmark = pytest.mark.gpu


def _tiny(tmp_path, dev):
    from test_gpu_decode import _tiny_model
    return _tiny_model(tmp_path, dev)[0]


def _ids(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def test_forward_batch_equals_forward_tree_of_each(dev, tmp_path):
    """Logits of a ragged batch behind a shared prompt against every sequence alone through the drafted path over a bf16
    cache. (A row's element may round to either side of a tie between the two.)"""
    ns = _tiny(tmp_path, dev)
    model, c = ns.model, ns.model.attn_config()
    prompt = [5, 17, 42, 7, 250, 3, 99, 1, 288]
    tails = [[12, 30, 31], [8], [77, 9], [30, 12, 4, 4, 4]]
    prefix = BatchKV(ns.cfg.n_layer, c, 1, 12, dev)
    for piece in (prompt[:4], prompt[4:]):
        model.forward_batch(_ids([piece], dev), prefix)
    assert prefix.pos.tolist() == [9] and prefix.length == 9
    kv = BatchKV(ns.cfg.n_layer, c, 4, 7, dev, prefix=prefix)
    n = 3
    first = _ids([(t[:n] + [0] * n)[:n] for t in tails], dev)
    counts = _ids([min(n, len(t)) for t in tails], dev)
    every = model.forward_batch(first, kv, counts, last_only=False)
    kv.reset()
    last = model.forward_batch(first, kv, counts)
    second = model.forward_batch(_ids([(t[n:] + [0, 0])[:2] for t in tails], dev), kv, _ids([max(0, len(t) - n) for t in tails], dev))
    assert kv.pos.tolist() == [len(t) for t in tails] and kv.length == 5
    for b, tail in enumerate(tails):
        one = DeviceKV(ns.cfg.n_layer, c, 40, dev, dtype=torch.bfloat16)
        draft = DraftKV(one, c, max_nodes=1)
        want = []
        for t in prompt + tail:
            want.append(model.forward_tree(_ids([t], dev), draft))
            commit(draft, _ids([0], dev), _ids([1], dev))
        want = torch.cat(want)[len(prompt):]
        m = min(n, len(tail))
        assert rel_max(to_np(every[b, :m]), to_np(want[:m])) < 2.0 ** -5
        assert rel_max(to_np(last[b]), to_np(want[m - 1])) < 2.0 ** -5
        if len(tail) > n:
            assert rel_max(to_np(second[b]), to_np(want[-1])) < 2.0 ** -5
    with pytest.raises(ValueError):
        model.forward_batch(first, kv)  # (7 rows hold no three more behind five)
    with pytest.raises(ValueError):
        model.forward_batch(first[:2], kv)


@pytest.mark.parametrize("t", ROWS)
def test_batch_of_one_prompt_in_any_cut(dev, tmp_path, t):
    """A prompt's rows and logits are the same, to rounding, whether it is a prefix, a sequence, or cut between."""
    ns = _tiny(tmp_path, dev)
    model, c = ns.model, ns.model.attn_config()
    ids = [5, 17, 42, 7, 250, 3, 99, 1, 288, 6, 6]
    whole = BatchKV(ns.cfg.n_layer, c, 1, 11, dev, dtype=t)
    want = model.forward_batch(_ids([ids], dev), whole)
    for cut in (1, 6, 10):
        prefix = BatchKV(ns.cfg.n_layer, c, 1, cut, dev, dtype=t)
        model.forward_batch(_ids([ids[:cut]], dev), prefix)
        kv = BatchKV(ns.cfg.n_layer, c, 2, 11 - cut, dev, dtype=t, prefix=prefix)
        got = model.forward_batch(_ids([ids[cut:]] * 2, dev), kv)
        assert rel_max(to_np(got), to_np(want.expand(2, -1))) < 2.0 ** -5
        k, _ = load_rows(whole, 0, cut, 11 - cut)
        assert rel_max(to_np(load_rows(kv, 0, 0, 11 - cut)[0]), to_np(k.expand(2, -1, -1, -1))) < 2.0 ** -5


def test_generate_batch(dev, tmp_path):
    ns = _tiny(tmp_path, dev)
    shared = [11, 200, 37, 5, 6, 7, 5]
    prompts = [shared + [9, 8], shared + [4], shared + [9, 8], shared + [1, 2, 3, 4]]
    steps = list(ns.generate_batch(prompts, max_tokens=12, stop_on_eos=False))
    assert len(steps) == 12 and all(len(s) == 4 and None not in s for s in steps)
    assert ns.stats.prompt_tokens == 7 + 2 + 1 + 2 + 4 and ns.stats.generated_tokens == 48
    assert [s[0] for s in steps] == [s[2] for s in steps]
    for b in (0, 1, 3):  # each as alone, over the same type of cache
        assert [s[b] for s in steps] == list(ns.generate(prompts[b], max_tokens=12, stop_on_eos=False, kv_dtype=torch.bfloat16))
    same = list(ns.generate_batch([shared] * 3, max_tokens=5))
    assert all(s[0] == s[1] == s[2] for s in same)
    assert list(ns.generate_batch([[3]], max_tokens=0)) == []
    for t in ROWS:
        runs = []
        for _ in range(2):
            torch.manual_seed(3)
            runs.append(list(ns.generate_batch([shared] * 5, max_tokens=6, temperature=30.0, top_k=30, min_p=0.01, kv_dtype=t)))
        assert runs[0] == runs[1] and len(runs[0]) == 6
        assert len({tuple(s[b] for s in runs[0]) for b in range(5)}) > 1  # (numbers of its own for every sequence)
    for bad in ([], [[1], []]):
        with pytest.raises(ValueError):
            list(ns.generate_batch(bad))
    with pytest.raises(NotImplementedError):
        list(ns.generate_batch(["text"]))
    with pytest.raises(ValueError):
        list(ns.generate_batch([[1]], min_p=2.0))


def test_generate_batch_ends(dev, tmp_path, monkeypatch):
    """A sequence ends with the context, or with the end-of-text token, and the others go on."""
    ns = _tiny(tmp_path, dev)
    prompts = [[5, 6, 7] * 3, [5, 6, 7, 9], [5, 6] + [4] * 16]
    steps = list(ns.generate_batch(prompts, max_tokens=30, stop_on_eos=False))
    small = dataclasses.replace(ns.model.attn_config(), context_length=20)
    monkeypatch.setattr(ns.model, "attn_config", lambda: small)
    cut = list(ns.generate_batch(prompts, max_tokens=30, stop_on_eos=False))
    for b, p in enumerate(prompts):
        mine = [s[b] for s in cut]
        assert mine[:21 - len(p)] == [s[b] for s in steps][:21 - len(p)] and mine[21 - len(p):] == [None] * (len(cut) - 21 + len(p))
    with pytest.raises(ValueError):
        list(ns.generate_batch([[5] * 21], max_tokens=2))
    monkeypatch.undo()
    piece = steps[3][1]  # the second sequence's fourth token ends it
    token = next(i for i in range(300) if ns._piece(i) == piece)
    monkeypatch.setitem(ns.gguf.metadata, "tokenizer.ggml.eos_token_id", token)
    got = list(ns.generate_batch(prompts, max_tokens=30))
    for b in range(3):
        want = [s[b] for s in steps]
        end = want.index(piece) if piece in want else 30
        assert [s[b] for s in got] == want[:end] + [None] * (len(got) - end)


def test_generate_with_more_filters(dev, tmp_path):
    """top_k=1 is greedy at any temperature, with drafts and without; the same seed gives the same tokens."""
    ns = _tiny(tmp_path, dev)
    want = list(ns.generate([11, 200, 37], max_tokens=15))
    assert list(ns.generate([11, 200, 37], max_tokens=15, temperature=1.5, top_k=1)) == want
    assert list(ns.generate([11, 200, 37], max_tokens=15, temperature=1.5, top_k=1, drafts=5)) == want
    assert list(ns.generate([11, 200, 37], max_tokens=15, temperature=1.5, min_p=1.0)) == want
    runs = []
    for _ in range(2):
        torch.manual_seed(5)
        runs.append(list(ns.generate([4, 5], max_tokens=10, temperature=1.2, top_k=20, top_p=0.9, min_p=0.02)))
    assert runs[0] == runs[1]
    for kw in (dict(top_k=-1), dict(min_p=1.5)):
        with pytest.raises(ValueError):
            list(ns.generate([4], temperature=1.0, **kw))
