"""Decoding with drafted tokens: several tokens per pass, checked against the target model's own distribution.

A pass takes a tree of up to 64 nodes (`MAX_NODES`): node 0 the sequence's last known token, the others drafts of what
may follow, each under its parent. `parents` (device int32) holds every node's parent, an earlier node; None is a
chain, which is also how a piece of a prompt goes through.
- `DraftKV`: the nodes' key and value rows, beside a `DeviceKV` (refused drafts never touch the cache);
- `tree_attn_qkv` / `tree_attn`: a layer's attention of the nodes over the cache and their ancestors, from the raw
  projections or from rotated queries and finished rows;
- `verify`: which nodes the target accepts, and the token that follows them;
- `commit`: the accepted nodes' rows into the caches, the position moved on;
- `LookupDrafts`: drafts looked up in the sequence itself (what followed its last tokens earlier), no second model.
The reference decodes one token per forward (api.py:193-237); these have no counterpart in it. Calls that share a
DraftKV (its rows and its workspace) must not overlap.
"""
from __future__ import annotations

import math

import torch

from .. import _native as N
from .decode import AttnConfig, DeviceKV, LayerViews

MAX_NODES = N.TREE_MAX_NODES


class DraftKV:
    """Key and value rows of up to max_nodes drafted tokens, [n_layer][n_kv][max_nodes][head_dim] in the cache's type
    (`k`, `v`: a view per layer), and the attention's workspace."""

    def __init__(self, kv: DeviceKV, cfg: AttnConfig, max_nodes: int = 16) -> None:
        if not 1 <= max_nodes <= MAX_NODES:
            raise ValueError(f"max_nodes {max_nodes}: 1 to {MAX_NODES}")
        n_layer, n_kv, _, head_dim = kv.k_stack.shape
        if (n_kv, head_dim) != (cfg.n_head_kv, cfg.head_dim):
            raise ValueError(f"a cache of {n_kv} heads of {head_dim} for a model with {cfg.n_head_kv} of {cfg.head_dim}")
        nb = N.load().nsx_tree_workspace_bytes(cfg.n_head, n_kv, head_dim, int(max_nodes), kv.ctx_max)
        if nb < 0:
            raise NotImplementedError(N.load().nsx_last_error().decode(errors="replace"))
        self.kv, self.max_nodes, self.heads = kv, int(max_nodes), (cfg.n_head, n_kv, head_dim)
        shape = (n_layer, n_kv, self.max_nodes, head_dim)
        self.k_stack = torch.zeros(shape, dtype=kv.dtype, device=kv.device)
        self.v_stack = torch.zeros(shape, dtype=kv.dtype, device=kv.device)
        self.k, self.v = LayerViews(self.k_stack), LayerViews(self.v_stack)
        self.workspace = torch.empty(nb, dtype=torch.uint8, device=kv.device)
        self._taken = torch.zeros(1, dtype=torch.int32, device=kv.device)  # commit's workgroups count themselves out here
        self._dt = N.act_dtype_code(kv.dtype)


def _check(name: str, t, dtype, device, numel: int | None = None) -> None:
    if t is None:
        return
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not {device}")
    if not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise ValueError(f"{name} must be contiguous{'' if numel is None else f' with {numel} elements'}, "
                         f"got {tuple(t.shape)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


# a device's current stream as an address: torch's own accessor where it has one, 0.1 us for the stream object's 2.9
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _call(what: str, fn, device: torch.device, *args) -> None:
    """fn(*args, the device's current stream), with the device current."""
    if device.index == torch.cuda.current_device():
        rc = fn(*args, _stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(device.index))
    if rc:
        N.check(rc, what)


def _stacked(kv: DeviceKV, draft: DraftKV) -> bool:
    """Whether the layers are still the views of the stacks that they were made as."""
    try:
        return (kv.k.stack is kv.k_stack and kv.v.stack is kv.v_stack and draft.k.stack is draft.k_stack
                and draft.v.stack is draft.v_stack)
    except AttributeError:  # lists of the caller's
        return False


def _tree(x: torch.Tensor, row: int, name: str, draft: DraftKV, layer: int, cfg: AttnConfig, sinks, parents, out):
    """Checks shared by both attention calls -> (nodes, out)."""
    kv = draft.kv
    if kv.length > kv.ctx_max:
        raise ValueError(f"kv.length {kv.length} lies past the cache's {kv.ctx_max} rows")
    N.require_device(x)
    n = x.numel() // row if x.dim() > 1 else 1
    _check(name, x, torch.float32, kv.k_stack.device, n * row)
    if not 1 <= n <= draft.max_nodes:
        raise ValueError(f"{n} nodes: this DraftKV holds 1 to {draft.max_nodes}")
    if (cfg.n_head, cfg.n_head_kv, cfg.head_dim) != draft.heads:
        raise ValueError(f"{cfg.n_head} query heads over {cfg.n_head_kv} of {cfg.head_dim}; the DraftKV was made for "
                         "{} over {} of {}".format(*draft.heads))
    if not 0 <= layer < len(draft.k):
        raise IndexError(f"layer {layer} of {len(draft.k)}")
    if not _stacked(kv, draft):  # a layer of the caller's: the kernels take its shape and type for granted
        for name, t, like in (("kv.k", kv.k, kv.k_stack), ("kv.v", kv.v, kv.v_stack), ("draft.k", draft.k, draft.k_stack),
                              ("draft.v", draft.v, draft.v_stack)):
            _check(f"{name}[{layer}]", t[layer], kv.dtype, x.device, like[layer].numel())
    _check("parents", parents, torch.int32, x.device, n)
    _check("sinks", sinks, torch.float32, x.device, cfg.n_head)
    _check("out", out, torch.float32, x.device, n * cfg.n_head * cfg.head_dim)
    if out is None:
        out = torch.empty((n, cfg.n_head, cfg.head_dim), dtype=torch.float32, device=x.device)
    return n, out


def tree_attn(q: torch.Tensor, cfg: AttnConfig, draft: DraftKV, layer: int, sinks: torch.Tensor | None, window: int,
              parents: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Sink attention of the nodes' rotated queries (n, n_head * head_dim) over the layer's cache (kv.pos rows) and the
    rows that draft.k / draft.v hold of their ancestors and themselves, the last `window` positions of those when
    window > 0 -> (n, n_head, head_dim) fp32. A device position outside 0 .. kv.ctx_max leaves the output unwritten; the
    host's mirror kv.length is checked."""
    n, y = _tree(q, cfg.n_head * cfg.head_dim, "q", draft, layer, cfg, sinks, parents, out)
    kv = draft.kv
    _call("tree_attn", N.load().nsx_tree_attn, q.device, q.data_ptr(), kv.k[layer].data_ptr(), kv.v[layer].data_ptr(),
          draft._dt, draft.k[layer].data_ptr(), draft.v[layer].data_ptr(), _ptr(parents), n, draft.max_nodes,
          _ptr(sinks), cfg.n_head, cfg.n_head_kv, cfg.head_dim, kv.pos.data_ptr(), kv.ctx_max, int(window),
          1.0 / math.sqrt(cfg.head_dim), draft.workspace.data_ptr(), draft.workspace.numel(), y.data_ptr())
    return y


def tree_attn_qkv(qkv: torch.Tensor, bq, bk, bv, cfg: AttnConfig, inv_freq: torch.Tensor, amp: float, draft: DraftKV,
                  layer: int, sinks: torch.Tensor | None, window: int, parents: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """tree_attn from the nodes' raw q | k | v projections (n, (n_head + 2 n_kv) * head_dim), left unchanged: bias and
    rotary at each node's position, its key and value rows (in the cache's type) into draft.k / draft.v."""
    d, dev = cfg.head_dim, qkv.device
    n, y = _tree(qkv, (cfg.n_head + 2 * cfg.n_head_kv) * d, "qkv", draft, layer, cfg, sinks, parents, out)
    for name, t, m in (("bq", bq, cfg.n_head * d), ("bk", bk, cfg.n_head_kv * d), ("bv", bv, cfg.n_head_kv * d),
                       ("inv_freq", inv_freq, d // 2)):
        _check(name, t, torch.float32, dev, m)
    kv = draft.kv
    _call("tree_attn_qkv", N.load().nsx_tree_attn_qkv, dev, qkv.data_ptr(), _ptr(bq), _ptr(bk), _ptr(bv),
          inv_freq.data_ptr(), float(amp), kv.k[layer].data_ptr(), kv.v[layer].data_ptr(), draft._dt,
          draft.k[layer].data_ptr(), draft.v[layer].data_ptr(), _ptr(parents), n, draft.max_nodes, _ptr(sinks),
          cfg.n_head, cfg.n_head_kv, d, kv.pos.data_ptr(), kv.ctx_max, int(window), 1.0 / math.sqrt(d),
          draft.workspace.data_ptr(), draft.workspace.numel(), y.data_ptr())
    return y


def commit(draft: DraftKV, path: torch.Tensor, count: torch.Tensor) -> None:
    """Rows path[0 .. count - 1] of every layer's nodes into the caches' rows kv.pos, kv.pos + 1, ..., then kv.pos +=
    count on the device (path, count: device int32, as `verify` returns them for one sequence). The host's kv.length
    is the caller's to move on, by the count once it is known there; a full cache by that mirror is refused, and rows past
    the cache's end by the device's position are not written (kv.pos then stops at the end). Layers that were replaced in kv.k, kv.v, draft.k or
    draft.v are refused: the rows move from stack to stack."""
    kv = draft.kv
    if not _stacked(kv, draft):
        raise ValueError("a layer of kv.k, kv.v, draft.k or draft.v was replaced: commit moves the rows of the stacks "
                         "that they were made as")
    if kv.length >= kv.ctx_max:
        raise ValueError(f"the cache's {kv.ctx_max} rows are taken (kv.length {kv.length})")
    N.require_device(path, count)
    _check("path", path, torch.int32, kv.k_stack.device)
    _check("count", count, torch.int32, path.device, 1)
    n_layer, n_kv, m, d = draft.k_stack.shape
    if not 1 <= path.numel() <= m:
        raise ValueError(f"a path of {path.numel()} nodes: 1 to {m}")
    _call("commit", N.load().nsx_tree_commit, path.device, kv.k_stack.data_ptr(), kv.v_stack.data_ptr(),
          draft.k_stack.data_ptr(), draft.v_stack.data_ptr(), draft._dt, n_layer, n_kv, d, path.numel(), m,
          path.data_ptr(), count.data_ptr(), kv.pos.data_ptr(), kv.ctx_max, draft._taken.data_ptr())


def verify(logits: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor | None = None, *,
           parents: torch.Tensor | None = None, draft_probs: torch.Tensor | None = None, temperature: float = 0.0,
           lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens the target model accepts -> (count (B,), path (B, n), token (B,)), int32 on the device.

    logits (n, vocab) or (B, n, vocab) fp32 / fp16 / bf16: row i the target's distribution behind node i. tokens (B, n)
    int32, node 0 the last known token; uniforms (B, n) fp32 in [0, 1) (not needed at temperature 0). From node 0 on, a
    drafted child is accepted with the probability that leaves the tokens distributed as softmax(logits / temperature)
    would draw them: drafts taken as they are, or, with draft_probs (B, n - 1, vocab) fp32, drawn from those (chains).
    Temperature 0 accepts the largest logit's token, the lowest index of equals. parents: (n,) for all sequences or
    (B, n); lengths (B,) int32: how many of its nodes each sequence has. count: nodes accepted, node 0 among them;
    path: their indices, then -1; token: what follows them (drawn with uniforms[:, 0]), -1 where there is none."""
    if logits.dim() not in (2, 3):
        raise ValueError(f"logits of shape {tuple(logits.shape)}: (n, vocab) or (B, n, vocab)")
    N.require_device(logits)
    dt = N.act_dtype_code(logits.dtype)
    x = logits if logits.dim() == 3 else logits[None]
    B, n, V = x.shape
    dev = x.device
    # rows may lie apart (a padded vocabulary), all by the same stride
    ld = x.stride(1) if n > 1 else x.stride(0) if B > 1 else V
    if V and (x.stride(2) != 1 or ld < V or (n > 1 and B > 1 and x.stride(0) != n * ld)):
        x = x.contiguous()
        ld = V
    _check("tokens", tokens, torch.int32, dev, B * n)
    _check("uniforms", uniforms, torch.float32, dev, B * n)
    _check("draft_probs", draft_probs, torch.float32, dev, B * (n - 1) * V)
    _check("lengths", lengths, torch.int32, dev, B)
    stride = 0
    if parents is not None:
        _check("parents", parents, torch.int32, dev, n if parents.dim() == 1 else B * n)
        stride = 0 if parents.dim() == 1 else n
        if draft_probs is not None:
            raise ValueError("draft probabilities go with chains (no parents)")
    temperature = float(temperature)
    if temperature != 0.0 and uniforms is None:
        raise ValueError("a temperature above 0 needs uniforms")
    count = torch.empty(B, dtype=torch.int32, device=dev)
    path = torch.empty((B, n), dtype=torch.int32, device=dev)
    token = torch.empty(B, dtype=torch.int32, device=dev)
    lib = N.load()
    nb = max(0, lib.nsx_verify_workspace_bytes(B, n, V))
    ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=dev)  # stream-ordered scratch, as the outputs
    _call("verify", lib.nsx_verify, dev, x.data_ptr(), dt, ld, B, n, V, tokens.data_ptr(), _ptr(parents), stride,
          _ptr(lengths), _ptr(uniforms), _ptr(draft_probs), temperature, count.data_ptr(), path.data_ptr(),
          token.data_ptr(), ws.data_ptr(), max(nb, 16))
    return count, path, token


class LookupDrafts:
    """Drafts for a sequence from the sequence itself: where its last `ngram` tokens (or fewer) stood before, what
    followed them there, the latest places first, merged into a tree."""

    PLACES = 4  # earlier places of the same tokens that a proposal follows

    def __init__(self, tokens, ngram: int = 3) -> None:
        if ngram < 1:
            raise ValueError(f"ngram {ngram}: at least 1")
        self.ngram = int(ngram)
        self.tokens: list[int] = []
        self._after: dict[tuple, list[int]] = {}  # the indices behind a run of tokens
        self.extend(tokens)

    def extend(self, tokens) -> None:
        for t in tokens:
            self.tokens.append(int(t))
            end = len(self.tokens)
            for g in range(1, min(self.ngram, end) + 1):
                self._after.setdefault(tuple(self.tokens[end - g:]), []).append(end)

    def propose(self, n_drafts: int, depth: int | None = None) -> tuple[list[int], list[int]]:
        """(tokens, parents) of a tree: node 0 the sequence's last token, then up to n_drafts drafts, each no deeper
        than `depth`."""
        seq, nodes, parents = self.tokens, [self.tokens[-1]], [-1]
        depth = n_drafts if depth is None else min(depth, n_drafts)
        places: list[int] = []
        for g in range(min(self.ngram, len(seq)), 0, -1):
            for at in reversed(self._after[tuple(seq[-g:])][-self.PLACES - 1:]):
                if at < len(seq) and at not in places and len(places) < self.PLACES:
                    places.append(at)
        child: dict[tuple[int, int], int] = {}
        tips = {at: 0 for at in places}  # level by level, so that no place takes every node
        for level in range(depth):
            for at, tip in list(tips.items()):
                if at + level >= len(seq):
                    del tips[at]
                    continue
                key = (tip, seq[at + level])
                if key not in child:
                    if len(nodes) > n_drafts:
                        return nodes, parents
                    child[key] = len(nodes)
                    nodes.append(key[1])
                    parents.append(tip)
                tips[at] = child[key]
        return nodes, parents


__all__ = ["LookupDrafts", "MAX_NODES", "DraftKV", "tree_attn", "tree_attn_qkv", "commit", "verify"]
