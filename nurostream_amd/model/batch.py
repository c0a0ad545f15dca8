"""Several sequences at once: answers to one prompt, or many users' prompts behind a shared one.

- `BatchKV`: key and value rows of n_seq sequences, in bf16 or quantised to 8 bits (int8 or e4m3 with a scale per row),
  each sequence with a length of its own in device memory; `prefix`, another BatchKV of one sequence, holds the rows that
  all of them share, which are kept and read once for all;
- `append_qkv`: the new tokens' rows into the cache and their queries, from the raw projections: bias, norms of query and
  key heads (Qwen3's; optional), rotation, rounding or quantisation in one pass;
- `batch_attn`: their attention over the prefix and their own rows;
- `store_rows` / `load_rows`: finished rows into the cache, and the values it holds back.

A step of a batch is append_qkv and batch_attn for every layer, then `BatchKV.advance`; nothing in it waits for the host,
and it can be captured into a graph. A prompt goes the same way, several tokens a step (into a prefix first, then into
the batches that are given it). The reference decodes one sequence (api.py:193-237); these have no counterpart in it.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from .. import _native as N
from .decode import AttnConfig, DeviceKV
from .draft import _call, _check, _ptr

X_TYPES = {torch.float32: N.DT_F32, torch.float16: N.DT_F16, torch.bfloat16: N.DT_BF16}
ROW_TYPES = {torch.bfloat16: N.DT_BF16, torch.int8: N.KV_INT8, torch.float8_e4m3fn: N.KV_E4M3}


class BatchKV:
    """Key and value rows of n_seq sequences, up to ctx_max each: `k_stack`, `v_stack` [n_layer][n_seq][n_kv][ctx_max]
    [head_dim] of dtype (bfloat16, int8 or float8_e4m3fn), for 8 bits `k_scale`, `v_scale` fp32 per row; `pos`, the rows that
    each sequence holds (device int32), and `length`, the host's bound on them. prefix: a BatchKV of one sequence whose rows
    stand before every sequence's own (its length counts when a call runs, so it may still grow between calls)."""

    def __init__(self, n_layer: int, cfg: AttnConfig, n_seq: int, ctx_max: int, device, dtype: torch.dtype = torch.bfloat16,
                 prefix: "BatchKV | None" = None) -> None:
        if dtype not in ROW_TYPES:
            raise TypeError(f"rows of {dtype}: bfloat16, int8 or float8_e4m3fn")
        if n_layer < 1 or not 1 <= n_seq < 65536 or not 1 <= ctx_max < 1 << 30:
            raise ValueError(f"{n_layer} layers of {n_seq} sequences of {ctx_max} rows: at least 1 each, fewer than 65536 "
                             "sequences and 2^30 rows")
        if cfg.head_dim not in (64, 128):
            raise NotImplementedError(f"head_dim {cfg.head_dim} (the kernels are written for 64 and 128)")
        self.device, self.dtype, self.n_seq, self.ctx_max = torch.device(device), dtype, int(n_seq), int(ctx_max)
        self.heads = (cfg.n_head_kv, cfg.head_dim)
        shape = (n_layer, self.n_seq, cfg.n_head_kv, self.ctx_max)
        self.k_stack = torch.zeros((*shape, cfg.head_dim), dtype=dtype, device=self.device)
        self.v_stack = torch.zeros_like(self.k_stack)
        self.k_scale = self.v_scale = None
        if dtype != torch.bfloat16:
            self.k_scale = torch.zeros(shape, dtype=torch.float32, device=self.device)
            self.v_scale = torch.zeros_like(self.k_scale)
        self.device = self.k_stack.device
        self.pos = torch.zeros(self.n_seq, dtype=torch.int32, device=self.device)
        self.length = 0
        self.prefix = prefix
        if prefix is not None:
            if prefix.n_seq != 1 or prefix.prefix is not None:
                raise ValueError("a prefix is one sequence without a prefix of its own")
            if (prefix.heads, prefix.dtype, prefix.device, prefix.k_stack.shape[0]) != (self.heads, dtype, self.device, n_layer):
                raise ValueError("a prefix has its batch's layers, heads, row type and device")
        self._kind, self._index = ROW_TYPES[dtype], self.k_stack.get_device()
        self._scratch: dict[tuple, int] = {}  # bytes of the attention's workspace by sizes
        self._layers: dict = {}

    def rows(self, layer: int):
        """A layer as the kernels take it (a reference to its nsx_kv_rows)."""
        got = self._layers.get(layer)
        if got is None:
            if not 0 <= layer < self.k_stack.shape[0]:
                raise IndexError(f"layer {layer} of {self.k_stack.shape[0]}")
            got = C.byref(N.KvRowsC(self.k_stack[layer].data_ptr(), self.v_stack[layer].data_ptr(),
                            None if self.k_scale is None else self.k_scale[layer].data_ptr(),
                            None if self.v_scale is None else self.v_scale[layer].data_ptr(), self.pos.data_ptr(), self.n_seq,
                            self.ctx_max))
            self._layers[layer] = got
        return got

    def __setattr__(self, name, value) -> None:
        if name in ("k_stack", "v_stack", "k_scale", "v_scale", "pos", "prefix") and "_layers" in self.__dict__:
            raise AttributeError(f"{name} stays the tensor that the cache was made with (copy into it instead)")
        super().__setattr__(name, value)

    def __getstate__(self):  # (a copy has tensors of its own: its layers' addresses are taken anew)
        return {k: v for k, v in self.__dict__.items() if k != "_layers"}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state, _layers={}, _index=state["k_stack"].get_device())

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_stack, self.v_stack, self.k_scale, self.v_scale)
                   if t is not None)

    def reset(self) -> None:
        self.pos.zero_()
        self.length = 0

    def advance(self, n: int = 1, counts: torch.Tensor | None = None) -> None:
        """After the last layer: n more rows in every sequence, or counts[b] (device int32, at most n each). `length` grows
        by n either way: where the sequences' real lengths are known on the host, it may be set to the largest."""
        if n < 0 or self.length + n > self.ctx_max:
            raise ValueError(f"{n} rows behind up to {self.length} of a cache of {self.ctx_max}")
        if counts is None:
            self.pos.add_(n)
        else:
            _check("counts", counts, torch.int32, self.device, self.n_seq)
            self.pos.add_(counts.clamp(0, n))
        self.length += n

    def copy_from(self, kv: "DeviceKV | BatchKV") -> None:
        """Every layer's rows of another cache in place of this one's: of a DeviceKV (its rows become those of every
        sequence), or of a BatchKV of as many sequences (or of one), in this cache's type. Reads the lengths on the host."""
        if getattr(kv, "prefix", None) is not self.prefix:
            raise ValueError("the rows stand behind another prefix")
        pos = kv.pos.tolist()
        if isinstance(kv, BatchKV):
            shape = (kv.k_stack.shape[0], *kv.heads)
        else:
            shape = (kv.k_stack.shape[0], kv.k_stack.shape[1], kv.k_stack.shape[3])
        if shape != (self.k_stack.shape[0], *self.heads) or len(pos) not in (1, self.n_seq) or kv.k_stack.device != self.device:
            raise ValueError("the caches differ in layers, heads, sequences or device")
        n = max(pos)
        if n > self.ctx_max:
            raise ValueError(f"{n} rows into a cache of {self.ctx_max}")
        for layer in range(shape[0]):
            if isinstance(kv, BatchKV):
                k, v = load_rows(kv, layer, 0, n, dtype=torch.float32)
            else:
                k, v = kv.k[layer][None, :, :n].contiguous(), kv.v[layer][None, :, :n].contiguous()
            if k.shape[0] != self.n_seq:
                k, v = (t.expand(self.n_seq, -1, -1, -1).contiguous() for t in (k, v))
            store_rows(k, v, self, layer, 0)
        self.pos.copy_(kv.pos.expand(self.n_seq))
        self.length = n


def _fits(t: torch.Tensor, dtype: torch.dtype, index: int, numel: int) -> bool:
    """What `_check` looks for on the GPU, in the least of the host's time."""
    return t.dtype is dtype and t.get_device() == index and t.numel() == numel and t.is_contiguous()


def _tokens(x: torch.Tensor, heads: int, name: str, kv: BatchKV, cfg: AttnConfig, counts) -> int:
    """Checks shared by the calls on tokens -> tokens per sequence."""
    index = kv._index
    if index < 0 or x.get_device() != index:
        N.require_device(x)
    if x.dtype not in X_TYPES:
        N.act_dtype_code(x.dtype)
    G, d = kv.heads
    if cfg.n_head_kv != G or cfg.head_dim != d or cfg.n_head % G:
        raise ValueError(f"{cfg.n_head} query heads over {cfg.n_head_kv} of {cfg.head_dim}; the cache was made for {G} of {d}")
    numel, row = x.numel(), kv.n_seq * heads * d
    n = numel // row
    if n < 1 or n * row != numel:
        raise ValueError(f"{name} of shape {tuple(x.shape)} for {kv.n_seq} sequences and rows of {heads * d}")
    if x.get_device() != index or not x.is_contiguous():
        _check(name, x, x.dtype, kv.device, numel)
    if counts is not None and not _fits(counts, torch.int32, index, kv.n_seq):
        _check("counts", counts, torch.int32, kv.device, kv.n_seq)
    if kv.length + n > kv.ctx_max:
        raise ValueError(f"{n} tokens behind up to {kv.length} rows of a cache of {kv.ctx_max}")
    return n


def append_qkv(qkv: torch.Tensor, bq, bk, bv, cfg: AttnConfig, inv_freq: torch.Tensor, amp: float, kv: BatchKV, layer: int, *,
               counts: torch.Tensor | None = None, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
               eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """The new tokens' rotated queries (n_seq, n, n_head, head_dim), in qkv's type, their key and value rows written behind
    each sequence's kv.pos rows (kv.pos stays: `BatchKV.advance` after the last layer).

    qkv (n_seq, n, (n_head + 2 n_kv) * head_dim) fp32 / fp16 / bf16, the raw q | k | v projections; biases, norm weights
    (head_dim) and inv_freq fp32. A query or key head, bias added, is divided by sqrt(mean(x^2) + eps) and multiplied by its
    norm's weights, where given, then rotated by its position times inv_freq (taken in 64 bits), times amp. counts (n_seq,)
    int32: how many of the n tokens a sequence has; the others' queries are zero, and they leave no rows. Rows past the
    cache's end by the device's position are not written; the host's kv.length is checked."""
    d, H, G = cfg.head_dim, cfg.n_head, cfg.n_head_kv
    n = _tokens(qkv, H + 2 * G, "qkv", kv, cfg, counts)
    index = kv._index
    f32, nq, nk = torch.float32, H * d, G * d
    if not ((bq is None or _fits(bq, f32, index, nq)) and (bk is None or _fits(bk, f32, index, nk)) and
            (bv is None or _fits(bv, f32, index, nk)) and _fits(inv_freq, f32, index, d // 2) and
            (q_norm is None or _fits(q_norm, f32, index, d)) and (k_norm is None or _fits(k_norm, f32, index, d))):
        for name, t, m in (("bq", bq, nq), ("bk", bk, nk), ("bv", bv, nk), ("inv_freq", inv_freq, d // 2), ("q_norm", q_norm, d),
                           ("k_norm", k_norm, d)):
            _check(name, t, f32, kv.device, m)
    if out is None:
        q = qkv.new_empty((kv.n_seq, n, H, d))
    else:
        _check("out", out, qkv.dtype, kv.device, kv.n_seq * n * H * d)
        q = out
    _call("append_qkv", N.load().nsx_append_qkv, kv.device, qkv.data_ptr(), X_TYPES[qkv.dtype], _ptr(bq), _ptr(bk), _ptr(bv),
          _ptr(q_norm), _ptr(k_norm), eps, inv_freq.data_ptr(), amp, H, G, d, n, _ptr(counts), kv.rows(layer), kv._kind,
          None if kv.prefix is None else kv.prefix.pos.data_ptr(), q.data_ptr())
    return q


def batch_attn(q: torch.Tensor, cfg: AttnConfig, kv: BatchKV, layer: int, sinks: torch.Tensor | None, window: int, *,
               counts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Sink attention of the new tokens' queries (n_seq, n, n_head, head_dim), as `append_qkv` gives them with their rows
    written -> the same shape and type: token j of a sequence sees the prefix, its sequence's rows and the new tokens up
    to itself, the last `window` positions of those when window > 0. out: not q's own memory. fp32 queries are taken with all their bits and weights
    of 24; weights are rounded to 16 bits beside fp16 queries, to 8 beside bf16 ones. Tokens that a sequence does not have
    (`counts`) give zeros."""
    d, H, G = cfg.head_dim, cfg.n_head, cfg.n_head_kv
    n, window, prefix = _tokens(q, H, "q", kv, cfg, counts), min(int(window), 2 ** 31 - 1), kv.prefix  # (past it: all rows)
    if sinks is not None and not _fits(sinks, torch.float32, kv._index, H):
        _check("sinks", sinks, torch.float32, kv.device, H)
    if window < 0:
        raise ValueError(f"window {window}")
    if out is None:
        y = q.new_empty((kv.n_seq, n, H, d))
    else:
        _check("out", out, q.dtype, kv.device, q.numel())
        y = out
    lib = N.load()
    nb = kv._scratch.get((H, n, window))  # (by sizes alone: the prefix is the one that the cache was made with)
    if nb is None:
        nb = lib.nsx_batch_attn_workspace_bytes(H, G, d, kv.n_seq, n, kv.ctx_max, 0 if prefix is None else prefix.ctx_max, window)
        if nb < 0:
            raise ValueError(f"{n} tokens of {kv.n_seq} sequences: too many for one call")
        kv._scratch[H, n, window] = nb
    # stream-ordered scratch, as the output
    ws = None if nb == 0 else torch.empty(nb, dtype=torch.uint8, device=kv.device)
    _call("batch_attn", lib.nsx_batch_attn, kv.device, q.data_ptr(), X_TYPES[q.dtype], kv.rows(layer),
          None if prefix is None else prefix.rows(layer), kv._kind, H, G, d, n, _ptr(counts), _ptr(sinks), window,
          1.0 / math.sqrt(d), _ptr(ws), nb, y.data_ptr())
    return y


def _first(start, kv: BatchKV, n: int) -> tuple[torch.Tensor | None, int]:
    """A run of rows' first one: (device array, 0) or (None, the host's number, checked)."""
    if isinstance(start, torch.Tensor):
        if not _fits(start, torch.int32, kv._index, kv.n_seq):
            _check("start", start, torch.int32, kv.device, kv.n_seq)
        return start, 0
    start = int(start)
    if start < 0 or start + n > kv.ctx_max:
        raise ValueError(f"rows {start} to {start + n} of a cache of {kv.ctx_max}")
    return None, start


def store_rows(k: torch.Tensor, v: torch.Tensor, kv: BatchKV, layer: int, start: int | torch.Tensor = 0) -> None:
    """Finished key and value rows (n_seq, n_kv, n, head_dim), fp32 / fp16 / bf16, into rows start .. start + n - 1 of every
    sequence, in the cache's type. start: one number, or device int32 (n_seq,), rows outside the cache then not written.
    kv.pos stays."""
    N.require_device(k, v)
    code = N.act_dtype_code(k.dtype)
    G, d = kv.heads
    if k.dim() != 4 or (k.shape[0], k.shape[1], k.shape[3]) != (kv.n_seq, G, d) or v.shape != k.shape:
        raise ValueError(f"rows of shape {tuple(k.shape)} and {tuple(v.shape)}: ({kv.n_seq}, {G}, n, {d})")
    _check("k", k, k.dtype, kv.device)
    _check("v", v, k.dtype, kv.device)
    first, start0 = _first(start, kv, k.shape[2])
    _call("store_rows", N.load().nsx_store_rows, kv.device, k.data_ptr(), v.data_ptr(), code, k.shape[2], _ptr(first), start0,
          G, d, kv.rows(layer), kv._kind)


def load_rows(kv: BatchKV, layer: int, start: int | torch.Tensor, n: int,
              dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v): the values that rows start .. start + n - 1 of every sequence stand for, (n_seq, n_kv, n, head_dim) of dtype
    (fp32 / fp16 / bf16). start as in `store_rows`; rows outside the cache give zeros."""
    code = X_TYPES[dtype] if dtype in X_TYPES else N.act_dtype_code(dtype)
    G, d = kv.heads
    if n < 0:
        raise ValueError(f"{n} rows")
    first, start0 = _first(start, kv, n)
    if kv._index < 0:
        N.require_device(kv.k_stack)
    k = torch.empty((kv.n_seq, G, n, d), dtype=dtype, device=kv.device)
    v = torch.empty_like(k)
    _call("load_rows", N.load().nsx_load_rows, kv.device, kv.rows(layer), kv._kind, G, d, _ptr(first), start0, n,
          k.data_ptr(), v.data_ptr(), code)
    return k, v


__all__ = ["BatchKV", "append_qkv", "batch_attn", "store_rows", "load_rows"]
