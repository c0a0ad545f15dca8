"""Refusals of the calls on several sequences (model/batch.py, model/sampling.py) that end on the host: the C ABI's checks
of sizes, types, alignment and workspaces, and the Python calls' checks of their tensors (CPU only)."""
from __future__ import annotations

import copy
import ctypes as C

import pytest
import torch

from nurostream_amd import _native as N
from nurostream_amd.model.batch import BatchKV, append_qkv, batch_attn, load_rows, store_rows
from nurostream_amd.model.decode import AttnConfig
from nurostream_amd.model.sampling import sample


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from nurostream_amd import build
        build.build()
    return N.load()


def _cfg(n_head=16, n_kv=2, head_dim=64):
    return AttnConfig(n_head=n_head, n_head_kv=n_kv, head_dim=head_dim, vocab_size=10, rope_base=150000.0,
                      context_length=4096)


A = 1 << 20  # an address that no check follows
FAR = 1 << 40


def _rows(**kw):
    a = dict(k=A, v=A, k_scale=A, v_scale=A, pos=A, n_seq=3, ctx_max=100)
    a.update(kw)
    return N.KvRowsC(*(a[n] for n, _ in N.KvRowsC._fields_))


def _append(lib, kv=None, **kw):
    a = dict(qkv=FAR, dt=N.DT_F32, qb=A, kb=A, vb=A, qn=A, kn=A, eps=1e-6, inv=A, amp=1.0, H=16, G=2, d=64, n=5, counts=None,
             kind=N.KV_INT8, prefix=None, out=A)
    a.update(kw)
    return lib.nsx_append_qkv(a["qkv"], a["dt"], a["qb"], a["kb"], a["vb"], a["qn"], a["kn"], a["eps"], a["inv"], a["amp"],
                              a["H"], a["G"], a["d"], a["n"], a["counts"], C.byref(kv or _rows()), a["kind"], a["prefix"],
                              a["out"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=7), N.ETYPE), (dict(kind=N.DT_F32), N.ETYPE), (dict(kind=N.DT_F16), N.ETYPE), (dict(kind=9), N.ETYPE),
    (dict(d=96), N.ENOTIMPL), (dict(d=256), N.ENOTIMPL), (dict(H=15), N.EINVAL), (dict(H=0), N.EINVAL), (dict(G=0), N.EINVAL),
    (dict(G=2048, H=4096), N.EINVAL), (dict(H=8192), N.EINVAL), (dict(n=-1), N.EINVAL), (dict(n=1 << 24), N.EINVAL),
    (dict(n=1 << 62), N.EINVAL), (dict(eps=-1.0), N.EINVAL), (dict(eps=float("nan")), N.EINVAL), (dict(qkv=None), N.EINVAL),
    (dict(out=None), N.EINVAL), (dict(inv=None), N.EINVAL), (dict(qkv=FAR + 4), N.EINVAL), (dict(out=A + 8), N.EINVAL),
    (dict(qn=A + 4), N.EINVAL), (dict(kb=A + 4), N.EINVAL), (dict(out=FAR + 16), N.EINVAL), (dict(n=0), N.OK)])
def test_append_checks(lib, kw, code):
    assert _append(lib, **kw) == code


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 4), dict(k_scale=None), dict(v_scale=None),
                                dict(k_scale=A + 2), dict(n_seq=0), dict(n_seq=65536), dict(ctx_max=0), dict(ctx_max=1 << 30),
                                dict(pos=None)])
def test_cache_checks(lib, kw):
    kv = _rows(**kw)
    assert _append(lib, kv) == N.EINVAL
    assert _attn(lib, kv=kv) == N.EINVAL
    if "pos" not in kw:  # (rows are moved by numbers of the caller's)
        assert lib.nsx_store_rows(A, A, N.DT_F32, 3, None, 0, 2, 64, C.byref(kv), N.KV_INT8, None) == N.EINVAL
        assert lib.nsx_load_rows(C.byref(kv), N.KV_INT8, 2, 64, None, 0, 3, A, A, N.DT_F32, None) == N.EINVAL
        assert _attn(lib, prefix=_rows(**{"n_seq": 1, **kw})) == N.EINVAL


def _attn(lib, **kw):
    a = dict(q=A, dt=N.DT_F32, kv=None, prefix=None, kind=N.KV_INT8, H=16, G=2, d=64, n=5, counts=None, sinks=None, window=0,
             scale=0.125, ws=A, wsb=1 << 40, out=A + (1 << 30))
    a.update(kw)
    return lib.nsx_batch_attn(a["q"], a["dt"], C.byref(a["kv"] or _rows(ctx_max=5000)), a["prefix"] and C.byref(a["prefix"]), a["kind"], a["H"],
                              a["G"], a["d"], a["n"], a["counts"], a["sinks"], a["window"], a["scale"], a["ws"], a["wsb"],
                              a["out"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=3), N.ETYPE), (dict(kind=0), N.ETYPE), (dict(d=32), N.ENOTIMPL), (dict(H=17), N.EINVAL), (dict(n=-2), N.EINVAL),
    (dict(n=1 << 23), N.EINVAL), (dict(window=-1), N.EINVAL), (dict(q=None), N.EINVAL), (dict(out=None), N.EINVAL),
    (dict(q=A + 8), N.EINVAL), (dict(out=A + 4), N.EINVAL), (dict(ws=None), N.EINVAL), (dict(scale=0.0), N.EINVAL), (dict(scale=-1.0), N.EINVAL),
    (dict(scale=float("nan")), N.EINVAL), (dict(scale=float("inf")), N.EINVAL), (dict(ws=A + 8), N.EINVAL),
    (dict(wsb=0), N.EINVAL), (dict(out=A), N.EINVAL), (dict(out=A + 2 * 5 * 16 * 64 * 4 - 16), N.EINVAL), (dict(n=0), N.OK)])
def test_attention_checks(lib, kw, code):
    assert _attn(lib, **kw) == code
    assert _attn(lib, prefix=_rows(n_seq=1), **kw) == code


def test_attention_prefix_is_one_sequence(lib):
    assert _attn(lib, prefix=_rows(n_seq=2)) == N.EINVAL


@pytest.mark.parametrize("kw,code", [
    (dict(dt=3), N.ETYPE), (dict(kind=0), N.ETYPE), (dict(d=32), N.ENOTIMPL), (dict(G=0), N.EINVAL), (dict(n=-1), N.EINVAL),
    (dict(n=1 << 31), N.EINVAL), (dict(n=1 << 28), N.EINVAL), (dict(start0=1 << 31), N.EINVAL), (dict(start0=-(1 << 31)), N.EINVAL),
    (dict(k=None), N.EINVAL), (dict(v=None), N.EINVAL), (dict(k=A + 8), N.EINVAL), (dict(n=0), N.OK)])
def test_rows_checks(lib, kw, code):
    a = dict(k=A, v=A, dt=N.DT_F32, n=3, start0=0, G=2, d=64, kind=N.KV_INT8)
    a.update(kw)
    kv = _rows()
    if code == N.OK:  # two outputs in one place
        assert lib.nsx_load_rows(C.byref(kv), N.KV_INT8, 2, 64, None, 0, 3, A, A + 512, N.DT_F32, None) == N.EINVAL
    assert lib.nsx_store_rows(a["k"], a["v"], a["dt"], a["n"], None, a["start0"], a["G"], a["d"], C.byref(kv), a["kind"],
                              None) == code
    assert lib.nsx_load_rows(C.byref(kv), a["kind"], a["G"], a["d"], None, a["start0"], a["n"], a["k"], a["v"], a["dt"],
                             None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(dt=5), N.ETYPE), (dict(B=-1), N.EINVAL), (dict(B=65536), N.EINVAL), (dict(V=0), N.EINVAL), (dict(V=(1 << 22) + 1, ld=1 << 23), N.EINVAL),
    (dict(ld=99), N.EINVAL), (dict(T=-1.0), N.EINVAL), (dict(T=1e-31), N.EINVAL), (dict(T=1e31), N.EINVAL), (dict(T=float("nan")), N.EINVAL),
    (dict(p=0.0), N.EINVAL), (dict(p=1.01), N.EINVAL), (dict(p=float("nan")), N.EINVAL), (dict(m=-0.1), N.EINVAL), (dict(m=1.1), N.EINVAL),
    (dict(m=float("nan")), N.EINVAL), (dict(k=-1), N.EINVAL), (dict(u=None), N.EINVAL), (dict(u=None, T=0.0, Ts=A), N.EINVAL),
    (dict(x=None), N.EINVAL), (dict(tok=None), N.EINVAL), (dict(ws=None), N.EINVAL), (dict(ws=A + 4), N.EINVAL), (dict(wsb=0), N.EINVAL),
    (dict(B=0), N.OK)])
def test_sample_checks(lib, kw, code):
    a = dict(x=A, dt=N.DT_F32, ld=100, B=2, V=100, u=A, T=1.0, p=0.9, m=0.1, k=5, Ts=None, tok=A, ws=A, wsb=1 << 40)
    a.update(kw)
    st = N.SamplingC(a["T"], a["p"], a["m"], a["k"], a["Ts"], None, None, None)
    assert lib.nsx_sample(a["x"], a["dt"], a["ld"], a["B"], a["V"], a["u"], C.byref(st), a["tok"], a["ws"], a["wsb"], None) == code
    if code == N.EINVAL and set(kw) <= {"p", "m", "k"}:  # arrays stand in for the numbers
        assert lib.nsx_sample(a["x"], a["dt"], a["ld"], a["B"], a["V"], a["u"], None, a["tok"], a["ws"], a["wsb"], None) == N.EINVAL


def test_cache_object():
    cfg = _cfg()
    with pytest.raises(TypeError):
        BatchKV(1, cfg, 2, 10, "cpu", dtype=torch.float16)
    for bad in ((0, 2, 10), (1, 0, 10), (1, 65536, 10), (1, 2, 0), (1, 2, 1 << 30)):
        with pytest.raises(ValueError):
            BatchKV(bad[0], cfg, bad[1], bad[2], "cpu")
    with pytest.raises(NotImplementedError):
        BatchKV(1, _cfg(head_dim=32), 2, 10, "cpu")
    prefix = BatchKV(2, cfg, 1, 20, "cpu", dtype=torch.int8)
    kv = BatchKV(2, cfg, 3, 10, "cpu", dtype=torch.int8, prefix=prefix)
    for other in (BatchKV(2, cfg, 2, 20, "cpu", dtype=torch.int8), kv, BatchKV(1, cfg, 1, 20, "cpu", dtype=torch.int8),
                  BatchKV(2, cfg, 1, 20, "cpu"), BatchKV(2, _cfg(n_kv=4), 1, 20, "cpu", dtype=torch.int8)):
        with pytest.raises(ValueError):
            BatchKV(2, cfg, 3, 10, "cpu", dtype=torch.int8, prefix=other)
    for name in ("k_stack", "v_scale", "pos", "prefix"):
        with pytest.raises(AttributeError):
            setattr(kv, name, getattr(kv, name))
    kv.rows(0)
    with pytest.raises(IndexError):
        kv.rows(2)
    twin = copy.deepcopy(kv)  # tensors of its own, and their addresses
    assert twin.rows(1)._obj.k == twin.k_stack[1].data_ptr() != kv.rows(1)._obj.k and twin.prefix.k_stack is not prefix.k_stack
    assert kv.nbytes() == 2 * 2 * 3 * 2 * 10 * (64 + 4)
    kv.advance(4)
    kv.advance(5, counts=torch.tensor([0, 9, 2], dtype=torch.int32))
    assert kv.pos.tolist() == [4, 9, 6] and kv.length == 9
    for call in (lambda: kv.advance(2), lambda: kv.advance(-1), lambda: kv.advance(1, counts=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()
    kv.reset()
    assert kv.pos.tolist() == [0, 0, 0] and kv.length == 0


def test_calls_refuse_cpu_tensors():
    """Product calls run on the GPU only."""
    cfg, f = _cfg(), torch.zeros
    kv = BatchKV(1, cfg, 2, 10, "cpu")
    for call in (lambda: append_qkv(f(2, 1, 20 * 64), None, None, None, cfg, f(32), 1.0, kv, 0),
                 lambda: batch_attn(f(2, 1, 16, 64), cfg, kv, 0, None, 0), lambda: store_rows(f(2, 2, 3, 64), f(2, 2, 3, 64), kv, 0),
                 lambda: load_rows(kv, 0, 0, 3), lambda: sample(f(2, 9), f(2))):
        with pytest.raises(N.NativeError):
            call()


def _as_device(monkeypatch):
    """The calls' checks of their tensors, on the CPU."""
    monkeypatch.setattr(N, "require_device", lambda *t: None)


def test_python_checks(monkeypatch):
    _as_device(monkeypatch)
    cfg, f = _cfg(), torch.zeros
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    kv = BatchKV(1, cfg, 2, 10, "cpu")
    x, inv, q, rows = f(2, 3, 20 * 64), f(32), f(2, 3, 16, 64), f(2, 2, 3, 64)
    app = lambda qkv=x, **kw: append_qkv(qkv, kw.pop("bq", None), None, None, kw.pop("cfg", cfg), kw.pop("inv", inv), 1.0, kv,  # noqa: E731
                                         kw.pop("layer", 0), **kw)
    att = lambda q=q, **kw: batch_attn(q, kw.pop("cfg", cfg), kv, kw.pop("layer", 0), kw.pop("sinks", None), kw.pop("window", 0), **kw)  # noqa: E731
    for error, calls in {
        ValueError: (lambda: app(f(2, 0, 20 * 64)), lambda: app(f(2, 3, 20 * 64 - 1)), lambda: app(f(2, 20 * 64, 3).transpose(1, 2)),
                     lambda: app(f(2, 11, 20 * 64)), lambda: app(cfg=_cfg(n_kv=4)), lambda: app(cfg=_cfg(n_head=15)),
                     lambda: app(inv=f(31)), lambda: app(bq=f(64)), lambda: app(q_norm=f(128)), lambda: app(counts=i32(3)),
                     lambda: app(out=f(2, 3, 15, 64)), lambda: att(f(2, 3, 16, 32)[..., :31]), lambda: att(sinks=f(15)),
                     lambda: att(window=-1), lambda: att(counts=i32(1)), lambda: att(out=f(1)), lambda: att(f(2, 11, 16, 64)),
                     lambda: store_rows(rows, rows[:1], kv, 0), lambda: store_rows(rows[:1], rows[:1], kv, 0),
                     lambda: store_rows(rows, rows, kv, 0, 8), lambda: store_rows(rows, rows, kv, 0, -1),
                     lambda: store_rows(rows.transpose(0, 1), rows.transpose(0, 1), kv, 0), lambda: store_rows(rows, rows, kv, 0, i32(1)),
                     lambda: load_rows(kv, 0, 8, 3), lambda: load_rows(kv, 0, 0, -1), lambda: sample(f(3), f(3)),
                     lambda: sample(f(2, 9), f(3)), lambda: sample(f(2, 9), f(2), top_p=f(3)), lambda: sample(f(2, 9), f(2), out=i32(1))),
        TypeError: (lambda: app(x.double()), lambda: app(x.to(torch.int8)), lambda: app(bq=f(16 * 64, dtype=torch.float16)),
                    lambda: app(counts=f(2)), lambda: app(out=q.half()), lambda: att(q.double()), lambda: att(out=q.half()),
                    lambda: store_rows(rows, rows.half(), kv, 0), lambda: store_rows(rows.double(), rows.double(), kv, 0),
                    lambda: load_rows(kv, 0, 0, 3, dtype=torch.int8), lambda: store_rows(rows, rows, kv, 0, f(2)),
                    lambda: sample(f(2, 9, dtype=torch.float64), f(2)), lambda: sample(f(2, 9), f(2), top_k=f(2)),
                    lambda: sample(f(2, 9), f(2).double())),
        IndexError: (lambda: load_rows(kv, 1, 0, 3), lambda: load_rows(kv, -1, 0, 3)),
    }.items():
        for n, call in enumerate(calls):
            with pytest.raises(error):
                call()
                pytest.fail(f"{error.__name__} call {n}")
    kv.length = 8  # the host's bound on the rows taken
    for call in (app, att):
        with pytest.raises(ValueError):
            call()


def test_copy_from_refusals():
    cfg = _cfg()
    prefix = BatchKV(1, cfg, 1, 9, "cpu")
    kv, other = BatchKV(1, cfg, 3, 9, "cpu", prefix=prefix), BatchKV(1, cfg, 3, 20, "cpu")
    with pytest.raises(ValueError):  # rows behind a prefix stand at other positions than rows behind none
        other.copy_from(kv)
    with pytest.raises(ValueError):
        kv.copy_from(other)
    with pytest.raises(ValueError):
        other.copy_from(BatchKV(1, cfg, 2, 9, "cpu"))
    with pytest.raises(ValueError):
        other.copy_from(BatchKV(2, cfg, 3, 9, "cpu"))
    other.pos.fill_(10)
    with pytest.raises(ValueError):
        BatchKV(1, cfg, 3, 9, "cpu").copy_from(other)


@pytest.mark.parametrize("top_k,top_p,min_p", [(5, 1.0, 0.0), (0, 0.7, 0.05), (12, 0.6, 0.01), (300, 0.95, 0.0), (1, 0.5, 0.9)])
def test_nucleus_keeps_what_sampling_may_draw(top_k, top_p, min_p):
    """generate's filter ahead of verification, against the definition written out."""
    from batch_cases import sample_exact
    from nurostream_amd.api import NeuroStream
    g = torch.Generator().manual_seed(top_k)
    lg = 3 * torch.randn(4, 200, generator=g)
    kept = NeuroStream._nucleus(lg, 0.8, top_p, top_k, min_p) > float("-inf")
    u = [(i + 0.5) / 4000 for i in range(4000)]
    each = lambda x: [x] * 4000  # noqa: E731
    for r in range(2):
        drawn = set(sample_exact(lg[r:r + 1].expand(4000, -1), u, each(0.8), each(top_k), each(top_p), each(min_p)))
        assert drawn <= set(kept[r].nonzero()[:, 0].tolist())
        heavy = torch.softmax(lg[r].double() / 0.8, -1) * kept[r]
        assert drawn >= set((heavy / heavy.sum() > 1 / 2000).nonzero()[:, 0].tolist())
