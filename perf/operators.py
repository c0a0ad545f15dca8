"""Decoding with drafted tokens, operator by operator: what is computed, at which sizes, in plain torch and through
the framework's calls.

Three operators:

- "attn": attention of a tree of drafted tokens (nodes) over a layer's cache and over each node's ancestors, with
  sinks and a sliding window. Form "qkv" takes the raw q | k | v projections (bias, rotary, the nodes' key and value
  rows kept beside the cache); form "rotated" takes finished queries and rows. A prompt in pieces is the same call
  with a chain for a tree.
- "verify": which drafted tokens the target model accepts, given random numbers, and the token that follows them.
- "commit": the accepted nodes' rows of every layer into the caches, and the position moved on.

`listed()` are fixed cases, `draw()` more of the same ranges. With `own` false, `run` computes the plain form.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
D = 64  # head dimension of the framework's attention
#: YaRN as this repository's decode benchmark sets it
ROPE = {"rope_base": 150000.0, "rope_factor": 32.0, "original_context": 4096, "beta_fast": 32.0, "beta_slow": 1.0}
VOCAB_A, VOCAB_B = 201088, 151936  # the repository's two LM heads
MAX_NODES = 64
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed() -> list[dict]:
    def attn(name, form, tree, nodes, n_head, n_kv, ctx, window, dtype):
        return {"name": name, "kind": "attn", "form": form, "tree": tree, "nodes": nodes, "n_head": n_head,
                "n_kv": n_kv, "ctx": ctx, "window": window, "dtype": dtype}

    def verify(name, batch, nodes, vocab, tree, q, temperature, ragged, dtype):
        return {"name": name, "kind": "verify", "batch": batch, "nodes": nodes, "vocab": vocab, "tree": tree, "q": q,
                "temperature": temperature, "ragged": ragged, "dtype": dtype}

    return [
        # one token early in a conversation over a 16-bit cache: the smallest call, launches and latency
        attn("attn_1_ctx203_bf16", "rotated", "chain", 1, 64, 8, 203, 0, "bfloat16"),
        # a sliding-window layer under a tree: few keys, most of them at the window's edge
        attn("attn_tree23_window128", "qkv", "tree", 23, 64, 8, 3001, 128, "float32"),
        # a few drafted tokens in a long conversation, fp32 cache
        attn("attn_tree16_ctx16384", "qkv", "tree", 16, 64, 8, 16384, 0, "float32"),
        # a piece of a prompt
        attn("attn_chain64_ctx6000", "qkv", "chain", 64, 64, 8, 6000, 0, "float32"),
        # a small tree over a very long half-precision cache, four query heads per kv head
        attn("attn_tree7_ctx131000_f16", "rotated", "tree", 7, 32, 8, 131000, 0, "float16"),
        # a full tree over a long bf16 cache: the largest
        attn("attn_tree64_ctx65536_bf16", "rotated", "tree", 64, 64, 8, 65536, 0, "bfloat16"),
        # greedy decoding, five drafted tokens in a row
        verify("verify_greedy_chain6", 1, 6, VOCAB_A, "chain", False, 0.0, False, "float32"),
        # sampling with a tree of looked-up drafts
        verify("verify_tree32", 1, 32, VOCAB_A, "tree", False, 0.8, False, "float32"),
        # a draft model's tokens with their probabilities, a small vocabulary
        verify("verify_q_chain5_v32001", 1, 5, 32001, "chain", True, 1.0, False, "float32"),
        # the same for a batch of sequences with differing numbers of drafts, bf16 logits
        verify("verify_q_batch24_bf16", 24, 5, VOCAB_B, "chain", True, 0.7, True, "bfloat16"),
        # the accepted path of a chain of 6 into the caches of 36 layers
        {"name": "commit_36_layers_n6", "kind": "commit", "layers": 36, "n_kv": 8, "nodes": 6, "ctx": 512,
         "dtype": "float32"},
        # a whole piece of a prompt
        {"name": "commit_24_layers_n64_bf16", "kind": "commit", "layers": 24, "n_kv": 8, "nodes": 64, "ctx": 700,
         "dtype": "bfloat16"},
    ]


def _log_between(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(("attn", "attn", "attn", "verify", "verify", "commit"))
    if kind == "attn":
        n_kv = rng.choice((1, 2, 4, 8))
        n_head = n_kv * rng.choice((1, 3, 4, 5, 8, 8, 16))
        form, dtype = rng.choice((("qkv", "float32"), ("rotated", "float32"), ("rotated", "float16"),
                                  ("rotated", "bfloat16")))
        nodes = _log_between(rng, 1, MAX_NODES)
        most = min(131072, 64 * 64 * 65536 // (nodes * n_head))
        return {"kind": "attn", "form": form, "tree": rng.choice(("tree", "tree", "chain")), "nodes": nodes,
                "n_head": n_head, "n_kv": n_kv, "ctx": _log_between(rng, 1, most),
                "window": rng.choice((0, 0, 0, 128, _log_between(rng, 1, 5000))), "dtype": dtype}
    if kind == "verify":
        q = rng.random() < 0.5
        vocab = _log_between(rng, 1000, VOCAB_A)
        nodes = _log_between(rng, 2 if q else 1, 8 if q else MAX_NODES)
        batch = min(_log_between(rng, 1, 64), max(1, 24 * 5 * VOCAB_B // (nodes * vocab)))
        return {"kind": "verify", "batch": batch, "nodes": nodes, "vocab": vocab,
                "tree": "chain" if q else rng.choice(("tree", "tree", "chain")), "q": q,
                "temperature": rng.choice((1.0, round(rng.uniform(0.3, 1.5), 2))) if q else
                rng.choice((0.0, 1.0, round(rng.uniform(0.3, 1.5), 2))),
                "ragged": rng.random() < 0.5, "dtype": rng.choice(tuple(TYPES))}
    return {"kind": "commit", "layers": rng.randint(1, 40), "n_kv": rng.choice((1, 2, 4, 8)),
            "nodes": _log_between(rng, 1, MAX_NODES), "ctx": rng.randint(64, 1000), "dtype": rng.choice(tuple(TYPES))}


# -- inputs ------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 1000003 % (1 << 62))
    return g


def _parents(case: dict, seed: int) -> list[int]:
    """A tree's parents, each before its children (several children here and there), or a chain's."""
    n = case["nodes"]
    if case["tree"] == "chain":
        return [i - 1 for i in range(n)]
    r = np.random.default_rng(int(seed) % (1 << 62))
    return [-1] + [int(r.integers(max(0, i - 6), i)) for i in range(1, n)]


def _lineage(parents: list[int]) -> tuple[np.ndarray, np.ndarray]:
    """(depth of each node, [i, j]: j is i or one of its ancestors)."""
    n = len(parents)
    depth, anc = np.zeros(n, dtype=np.int64), np.eye(n, dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            depth[i] = depth[p] + 1
            anc[i] |= anc[p]
    return depth, anc


def _inv_freq() -> tuple[torch.Tensor, float]:
    """YaRN's inverse frequencies and amplitude."""
    half, base, factor = D // 2, ROPE["rope_base"], ROPE["rope_factor"]
    dims = torch.arange(half, dtype=torch.float32)
    inv = 1.0 / base ** (dims / half)
    turn = lambda n: D * math.log(ROPE["original_context"] / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(turn(ROPE["beta_fast"]), 0), min(turn(ROPE["beta_slow"]), D - 1)
    ramp = ((dims - low) / (high - low)).clamp(0, 1)
    return (inv * (1 - ramp) + inv / factor * ramp).to(DEVICE), 1 + 0.1 * math.log(factor)


def _attn_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    H, G, N, ctx, t = case["n_head"], case["n_kv"], case["nodes"], case["ctx"], TYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    s = {"case": case, "k": (normal(G, ctx, D) * 1.5).to(t), "v": normal(G, ctx, D).to(t), "sinks": normal(H)}
    s["parents"] = torch.tensor(_parents(case, seed), dtype=torch.int32, device=DEVICE)
    if case["form"] == "qkv":
        s["qkv"] = normal(N, (H + 2 * G) * D) * 1.5
        s["bq"], s["bk"], s["bv"] = (normal(n * D) * 0.1 for n in (H, G, G))
        s["inv"], s["amp"] = _inv_freq()
    else:
        s["q"] = normal(N, H * D) * 1.5
        s["dk"], s["dv"] = (normal(G, N, D) * 1.5).to(t), normal(G, N, D).to(t)
    return s


def _verify_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    B, N, V = case["batch"], case["nodes"], case["vocab"]
    rand = lambda *shape: torch.rand(*shape, generator=g, device=DEVICE)  # noqa: E731
    s = {"case": case, "parent_list": _parents(case, seed)}
    s["parents"] = torch.tensor(s["parent_list"], dtype=torch.int32, device=DEVICE)
    # an LM head's logits: a broad bulk and a few candidates far above it
    logits = 2.0 * torch.randn(B, N, V, generator=g, device=DEVICE)
    top = torch.randint(0, V, (B, N, 6), generator=g, device=DEVICE)
    logits.scatter_add_(2, top, 6 + 8 * rand(B, N, 6))
    s["logits"] = logits.to(TYPES[case["dtype"]])
    T = case["temperature"]
    tokens = torch.randint(0, V, (B, N), generator=g, device=DEVICE)
    s["probs"] = None
    if case["q"]:
        # a draft model that mostly agrees: its tokens are drawn from its own probabilities
        dl = logits[:, :N - 1] / (T or 1.0) + 0.5 * torch.randn(B, N - 1, V, generator=g, device=DEVICE)
        noise = -torch.log(-torch.log(rand(B, N - 1, V).clamp(1e-20, 1 - 1e-7)))
        tokens[:, 1:] = (dl + noise).argmax(-1)
        s["probs"] = torch.softmax(dl, -1)
    elif N > 1:
        # looked-up drafts: a node's children are its likeliest tokens, one in eight is anything
        best = s["logits"].float().topk(min(8, V), -1).indices
        rank, seen = [], {}
        for p in s["parent_list"][1:]:
            rank.append(seen.get(p, 0) % best.shape[-1])
            seen[p] = seen.get(p, 0) + 1
        pick = best[:, torch.tensor(s["parent_list"][1:], device=DEVICE), torch.tensor(rank, device=DEVICE)]
        tokens[:, 1:] = torch.where(rand(B, N - 1) < 0.125, tokens[:, 1:], pick)
    s["tokens"] = tokens.to(torch.int32)
    s["u"] = rand(B, N)
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, N + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
    return s


def _commit_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    L, G, N, ctx, t = case["layers"], case["n_kv"], case["nodes"], case["ctx"], TYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE).to(t)  # noqa: E731
    s = {"case": case, "k": normal(L, G, ctx, D), "v": normal(L, G, ctx, D), "dk": normal(L, G, N, D),
         "dv": normal(L, G, N, D)}
    r = np.random.default_rng(int(seed) % (1 << 62))
    count = int(r.integers((N + 1) // 2, N + 1))  # the path takes at least half of the nodes
    path = np.full(N, -1, dtype=np.int64)
    path[:count] = np.concatenate([[0], 1 + np.sort(r.choice(N - 1, count - 1, replace=False))]) if N > 1 else [0]
    s["path"] = torch.tensor(path, dtype=torch.int32, device=DEVICE)
    s["count"] = torch.tensor([count], dtype=torch.int32, device=DEVICE)
    s["pos"] = torch.tensor([int(r.integers(0, max(1, ctx - N)))], dtype=torch.int32, device=DEVICE)
    return s


def prepare(case: dict, seed: int) -> dict:
    s = {"attn": _attn_inputs, "verify": _verify_inputs, "commit": _commit_inputs}[case["kind"]](case, seed)
    if own and case["kind"] != "verify":
        _own_caches(case, s)
    return s


def _own_caches(case: dict, s: dict) -> None:
    """The cache and the drafts' rows as a user's program holds them."""
    from nurostream_amd.model.decode import AttnConfig, DeviceKV
    from nurostream_amd.model.draft import DraftKV

    attn = case["kind"] == "attn"
    n_layer, G, ctx, N = 1 if attn else case["layers"], case["n_kv"], case["ctx"], case["nodes"]
    cfg = AttnConfig(n_head=case["n_head"] if attn else G, n_head_kv=G, head_dim=D, vocab_size=VOCAB_A,
                     context_length=131072, sliding_window=128, **ROPE)
    kv = DeviceKV(n_layer, cfg, ctx, DEVICE, dtype=TYPES[case["dtype"]])
    draft = DraftKV(kv, cfg, max_nodes=N)
    for layer in range(n_layer):
        kv.k[layer].copy_(s["k"] if attn else s["k"][layer])
        kv.v[layer].copy_(s["v"] if attn else s["v"][layer])
        if "dk" in s:
            draft.k[layer].copy_(s["dk"] if attn else s["dk"][layer])
            draft.v[layer].copy_(s["dv"] if attn else s["dv"][layer])
    if attn:
        kv.pos.fill_(ctx)
        kv.length = ctx
    for name in ("k", "v", "dk", "dv"):
        s.pop(name, None)
    s["cfg"], s["kv"], s["draft"] = cfg, kv, draft


# -- one pass ----------------------------------------------------------------


def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        return {"attn": _attn_own, "verify": _verify_own, "commit": _commit_own}[kind](state)
    return {"attn": _attn_plain, "verify": _verify_plain, "commit": _commit_plain}[kind](state)


def _attn_own(s: dict):
    from nurostream_amd.model.draft import tree_attn, tree_attn_qkv

    case, draft = s["case"], s["draft"]
    if case["form"] == "qkv":
        out = tree_attn_qkv(s["qkv"], s["bq"], s["bk"], s["bv"], s["cfg"], s["inv"], s["amp"], draft, 0, s["sinks"],
                            case["window"], parents=s["parents"])
        return out, draft.k[0], draft.v[0]
    return (tree_attn(s["q"], s["cfg"], draft, 0, s["sinks"], case["window"], parents=s["parents"]),)


def _tree_of(parents: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(depth, ancestor-or-self matrix) of a parent list on the device: paths doubled until the longest is covered."""
    n = parents.numel()
    one = torch.eye(n, device=parents.device)
    step = (parents[:, None] == torch.arange(n, device=parents.device)[None, :]).float()
    anc = one + step
    for _ in range(max(1, (n - 1).bit_length())):
        anc = ((anc @ anc) > 0).float()
    return anc.sum(1) - 1, anc > 0


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Halves (a, b) of each head to (a cos - b sin, b cos + a sin); x: (N, heads, D), cos and sin: (N, 1, D / 2)."""
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _attn_plain(s: dict):
    case = s["case"]
    H, G, N, ctx, window = case["n_head"], case["n_kv"], case["nodes"], case["ctx"], case["window"]
    depth, anc = _tree_of(s["parents"])
    if case["form"] == "qkv":
        x = s["qkv"].reshape(N, H + 2 * G, D)
        # the angle is the 32-bit product of position and frequency, as the cache's keys were rotated
        angle = ((ctx + depth)[:, None] * s["inv"][None, :]).double()
        cos, sin = ((f(angle) * s["amp"]).float()[:, None] for f in (torch.cos, torch.sin))
        q = _rotate(x[:, :H] + s["bq"].reshape(H, D), cos, sin)
        dk = _rotate(x[:, H:H + G] + s["bk"].reshape(G, D), cos, sin).transpose(0, 1).contiguous()
        dv = (x[:, H + G:] + s["bv"].reshape(G, D)).transpose(0, 1).contiguous()
    else:
        q, dk, dv = s["q"].reshape(N, H, D), s["dk"].float(), s["dv"].float()
    first = max(0, ctx + 1 - window) if window else 0
    keys = torch.cat([s["k"][:, first:].float(), dk], 1)
    vals = torch.cat([s["v"][:, first:].float(), dv], 1)
    seen = torch.cat([torch.ones(N, ctx - first, dtype=torch.bool, device=q.device), anc], 1)
    if window:
        at = torch.cat([torch.arange(first, ctx, device=q.device), ctx + depth])
        seen = seen & ((ctx + depth)[:, None] - at[None, :] < window)
    qh = q.reshape(N, G, H // G, D).permute(1, 0, 2, 3).reshape(G, N * (H // G), D)
    score = torch.matmul(qh, keys.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(D))
    score = score.masked_fill_(~seen.repeat_interleave(H // G, 0)[None], -math.inf)
    sink = s["sinks"].reshape(G, 1, H // G).expand(G, N, H // G).reshape(G, -1, 1)
    top = torch.maximum(score.amax(-1, keepdim=True), sink)
    w = torch.exp_(score.sub_(top))
    out = torch.matmul(w, vals) / (w.sum(-1, keepdim=True) + torch.exp(sink - top))
    out = out.reshape(G, N, H // G, D).permute(1, 0, 2, 3).reshape(N, H, D)
    return (out, dk, dv) if case["form"] == "qkv" else (out,)


def _verify_own(s: dict):
    from nurostream_amd.model.draft import verify

    return verify(s["logits"], s["tokens"], s["u"], parents=s["parents"] if s["case"]["tree"] == "tree" else None,
                  draft_probs=s["probs"], temperature=s["case"]["temperature"], lengths=s["lengths"])


def _verify_plain(s: dict):
    case = s["case"]
    B, N, V = s["logits"].shape
    tok, par, dev = s["tokens"].long(), s["parent_list"], s["tokens"].device
    rows = torch.arange(B, device=dev)
    length = torch.full((B,), N, device=dev) if s["lengths"] is None else s["lengths"].long()
    cur = torch.zeros(B, dtype=torch.long, device=dev)
    taken = torch.zeros(B, N, dtype=torch.bool, device=dev)
    taken[:, 0] = length > 0
    if case["temperature"] == 0.0:
        lg = s["logits"].float()
        ids = torch.arange(V, device=dev)
        best = torch.where(lg == lg.amax(-1, keepdim=True), ids, V).amin(-1)
        for i in range(1, N):
            ok = (cur == par[i]) & (i < length) & (tok[:, i] == best[rows, cur])
            taken[:, i] = ok
            cur = torch.where(ok, i, cur)
        nxt = best[rows, cur]
    else:
        # in 64 bits: a long sum is compared with a random number
        x = s["logits"].double() / case["temperature"]
        w = torch.exp(x - x.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        left = torch.ones(B, dtype=torch.float64, device=dev)
        out = torch.zeros(B, N, dtype=torch.bool, device=dev)  # refused children of the current node
        for i in range(1, N):
            at = (cur == par[i]) & (i < length)
            p = w[rows, par[i], tok[:, i]]
            if s["probs"] is not None:
                ok = at & (s["u"][:, i].double() * s["probs"][rows, i - 1, tok[:, i]].double() < p)
            else:
                p = torch.where((out & (tok == tok[:, i:i + 1])).any(1), 0.0, p)
                ok = at & (s["u"][:, i].double() * left < p)
            taken[:, i] = ok
            left = torch.where(ok, 1.0, torch.where(at, left - p, left))
            out = out & ~ok[:, None]
            out[:, i] = at & ~ok
            cur = torch.where(ok, i, cur)
        w = w[rows, cur]
        refused = out.any(1, keepdim=True)
        if s["probs"] is not None:
            q = s["probs"][rows, cur.clamp(max=N - 2)].double()
            w = torch.where(refused, (w - q).clamp_(min=0.0), w)
        else:
            gone = torch.zeros(B, V + 1, dtype=torch.bool, device=dev)
            gone.scatter_(1, torch.where(out, tok, V), True)
            w = w.masked_fill(gone[:, :V], 0.0)
        mass = w.cumsum(-1)
        nxt = (mass <= s["u"][:, :1].double() * mass[:, -1:]).sum(-1).clamp_(max=V - 1)
    count = taken.sum(1)
    order = torch.where(taken, torch.arange(N, device=dev), N).sort(1).values
    path = torch.where(order < N, order, -1)
    return count.to(torch.int32), path.to(torch.int32), torch.where(length > 0, nxt, -1).to(torch.int32)


def _commit_own(s: dict):
    from nurostream_amd.model.draft import commit

    kv = s["kv"]
    kv.pos.copy_(s["pos"])  # the same place in the cache every pass
    commit(s["draft"], s["path"], s["count"])
    return kv.k_stack, kv.v_stack, kv.pos


def _commit_plain(s: dict):
    case, n = s["case"], s["path"].numel()
    j = torch.arange(n, device=DEVICE)
    at = s["pos"].long() + j
    keep = (j < s["count"])[None, None, :, None]
    at = at.clamp(max=case["ctx"] - 1)
    src = s["path"].long().clamp(min=0)
    for cache, rows in ((s["k"], s["dk"]), (s["v"], s["dv"])):
        cache[:, :, at] = torch.where(keep, rows[:, :, src], cache[:, :, at])
    return s["k"], s["v"], s["pos"] + s["count"]


# -- what a pass cannot do without -------------------------------------------


def _visible(case: dict) -> tuple[int, int]:
    """(cache rows that some node sees, sum over the nodes of the keys each sees), a tree taken as a chain."""
    N, ctx, window = case["nodes"], case["ctx"], case["window"]
    if not window:
        return ctx, N * ctx + N * (N + 1) // 2
    seen = [min(window, ctx + i + 1) for i in range(N)]
    return max(0, min(ctx, window - 1)), sum(seen)


def work(case: dict) -> dict:
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    if case["kind"] == "attn":
        H, G, N, es = case["n_head"], case["n_kv"], case["nodes"], size[case["dtype"]]
        rows, pairs = _visible(case)
        io = N * H * D * 4 * 2 + 2 * N * G * D * (es + (4 if case["form"] == "qkv" else 0))
        return {"bytes": 2 * rows * G * D * es + io, "flops": 4 * D * H * pairs}
    if case["kind"] == "verify":
        B, N, V = case["batch"], case["nodes"], case["vocab"]
        return {"bytes": B * N * V * size[case["dtype"]] + (B * V * 4 if case["q"] else 0), "flops": 2 * B * N * V}
    moved = case["layers"] * 2 * case["n_kv"] * D * size[case["dtype"]] * (3 * case["nodes"] // 4 + 1)
    return {"bytes": 2 * moved, "flops": 0}


# -- the definition in 64 bits -----------------------------------------------


def exact(case: dict, seed: int):
    if case["kind"] == "attn":
        return _attn_exact(case, _attn_inputs(case, seed))
    if case["kind"] == "verify":
        return _verify_exact(case, _verify_inputs(case, seed))
    return _commit_exact(_commit_inputs(case, seed))


def _attn_exact(case: dict, s: dict):
    """Node by node, each over the keys that it sees."""
    H, G, N, ctx, window = case["n_head"], case["n_kv"], case["nodes"], case["ctx"], case["window"]
    R = H // G
    depth, anc = _lineage(s["parents"].tolist())
    if case["form"] == "qkv":
        x = s["qkv"].double().reshape(N, H + 2 * G, D)
        q, dk, dv = x[:, :H] + s["bq"].double().reshape(H, D), x[:, H:H + G] + s["bk"].double().reshape(G, D), \
            x[:, H + G:] + s["bv"].double().reshape(G, D)
        for i in range(N):
            angle = (torch.tensor(float(ctx + depth[i]), device=DEVICE) * s["inv"]).double()
            turn = torch.polar(torch.full_like(angle, s["amp"]), angle)
            for rows in (q, dk):
                z = torch.complex(rows[i, :, :D // 2].clone(), rows[i, :, D // 2:].clone()) * turn
                rows[i] = torch.cat([z.real, z.imag], -1)
    else:
        q, dk, dv = s["q"].double().reshape(N, H, D), s["dk"].double().transpose(0, 1), s["dv"].double().transpose(0, 1)
    out = torch.empty(N, H, D, dtype=torch.float64, device=DEVICE)
    for g in range(G):
        k, v = s["k"][g].double(), s["v"][g].double()
        for i in range(N):
            lo = max(0, ctx + int(depth[i]) + 1 - window) if window else 0
            kin = [j for j in range(N) if anc[i, j] and (not window or depth[i] - depth[j] < window)]
            keys, vals = torch.cat([k[lo:], dk[kin, g]]), torch.cat([v[lo:], dv[kin, g]])
            heads = slice(g * R, (g + 1) * R)
            sc = torch.cat([q[i, heads] @ keys.T.contiguous() / math.sqrt(D), s["sinks"][heads].double()[:, None]], 1)
            out[i, heads] = torch.softmax(sc, -1)[:, :-1] @ vals
    if case["form"] != "qkv":
        return (out,)
    return out, dk.transpose(0, 1).contiguous(), dv.transpose(0, 1).contiguous()


def _verify_exact(case: dict, s: dict):
    """Sequence by sequence on the host, reading only the rows of the nodes that are reached."""
    B, N, V = s["logits"].shape
    T, par, tok, u = case["temperature"], s["parent_list"], s["tokens"].cpu().numpy(), s["u"].cpu().numpy()
    lengths = [N] * B if s["lengths"] is None else s["lengths"].tolist()
    counts, paths, nexts = [], [], []
    for b in range(B):
        path, nxt = [], -1
        if lengths[b] > 0:
            path, i = [0], 0
            while True:
                row = s["logits"][b, path[-1]].double().cpu().numpy()
                if T == 0.0:
                    prob = np.zeros(V)
                    prob[int(np.argmax(row))] = 1.0
                else:
                    prob = np.exp((row - row.max()) / T)
                    prob /= prob.sum()
                child, went = [c for c in range(path[-1] + 1, lengths[b]) if par[c] == path[-1]], False
                for c in child:
                    x, total = int(tok[b, c]), prob.sum()
                    if s["probs"] is not None:
                        qrow = s["probs"][b, path[-1]].double().cpu().numpy()
                        went = float(u[b, c]) * qrow[x] < prob[x]
                        if not went:
                            prob = np.maximum(prob - qrow, 0.0)
                    else:
                        went = float(u[b, c]) * total < prob[x]
                        if not went:
                            prob[x] = 0.0
                    if went:
                        path.append(c)
                        break
                if not went:
                    break
            mass = np.cumsum(prob)
            nxt = min(int(np.searchsorted(mass, (0.0 if T == 0.0 else float(u[b, 0])) * mass[-1], side="right")), V - 1)
        counts.append(len(path))
        paths.append(path + [-1] * (N - len(path)))
        nexts.append(nxt)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return as_int(counts), as_int(paths), as_int(nexts)


def _commit_exact(s: dict):
    """Row by row."""
    pos, count, path = int(s["pos"]), int(s["count"]), s["path"].tolist()
    k, v = s["k"].double(), s["v"].double()
    for j in range(count):
        k[:, :, pos + j], v[:, :, pos + j] = s["dk"][:, :, path[j]].double(), s["dv"][:, :, path[j]].double()
    return k, v, s["pos"] + count
