"""Log-probability and embedding entry points without a GPU: argument errors come back
as statuses before anything touches a device, workspace sizes, and a replay of how
zs_logprobs finds the top alternatives from one key per thread."""

import ctypes as C

import numpy as np
import pytest

from zeninfer_b200 import _native

BAD = 1  # ZS_ERR_INVALID_ARGUMENT
F32, F16, BF16 = 0, 1, 2
P = 0x10000  # an aligned address; nothing dereferences it when the call is refused


@pytest.fixture(scope="module")
def lib():
    from zeninfer_b200 import build
    build.build_sampler()
    return _native.lib()


@pytest.fixture
def handle():
    import torch
    if torch.cuda.is_available():
        pytest.skip("refusals with a stand-in handle are for machines without a device")
    buf = C.create_string_buffer(1 << 16)
    yield C.cast(buf, C.c_void_p)


def _logprobs(lib, h, logits=P, dtype=F32, ld=100, batch=2, n=100, temp=1.0, row_temp=None, ids=P,
              ids_ld=1, m=1, logp=P, topn=4, tids=P, tlogp=P, ent=P, lse=P, rows=P):
    return lib.zs_logprobs(h, logits, dtype, ld, batch, n, temp, row_temp, ids, ids_ld, m, logp,
                           topn, tids, tlogp, ent, lse, rows, None)


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(logits=P + 2), dict(dtype=3), dict(dtype=-1), dict(ld=99),
    dict(batch=-1), dict(n=0), dict(n=-5), dict(temp=float("nan")), dict(row_temp=P + 1),
    dict(ids=None), dict(ids=P + 2), dict(ids_ld=0), dict(m=-1), dict(m=257), dict(logp=None),
    dict(logp=P + 1), dict(topn=-1), dict(topn=129), dict(tids=None), dict(tlogp=None),
    dict(tids=P + 2), dict(ent=P + 2), dict(lse=P + 3), dict(rows=P + 8), dict(ld=(1 << 40) + 1),
    dict(dtype=F16, logits=P + 1), dict(dtype=BF16, logits=P + 1),
])
def test_logprobs_refuses(lib, handle, change):
    assert _logprobs(lib, handle, **change) == BAD
    assert lib.zs_last_error()


def test_logprobs_null_handle_and_empty_batch(lib, handle):
    assert _logprobs(lib, None) == BAD
    assert _logprobs(lib, handle, batch=0, logits=None) == 0


def _backward(lib, h, logits=P, dtype=F32, ld=100, batch=2, n=100, rows=P, ids=P, ids_ld=1, m=1,
              gl=P, gh=P, gz=P, out=2 * P, gld=100):
    return lib.zs_logprobs_backward(h, logits, dtype, ld, batch, n, rows, ids, ids_ld, m, gl, gh,
                                    gz, out, gld, None)


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(dtype=9), dict(ld=10), dict(batch=-1), dict(n=0), dict(rows=None),
    dict(rows=P + 4), dict(ids=None), dict(ids_ld=0), dict(m=300), dict(gl=None), dict(gl=P + 1),
    dict(gh=P + 2), dict(gz=P + 2), dict(out=None), dict(out=P + 2), dict(gld=99),
    dict(out=P, ld=128, gld=104), dict(gld=(1 << 40) + 1), dict(batch=1 << 30, n=1 << 20, ld=1 << 20, gld=1 << 20),
])
def test_backward_refuses(lib, handle, change):
    assert _backward(lib, handle, **change) == BAD


def _lmhead(lib, h, hidden=P, hld=64, norm=P, w=P, batch=4, E=64, V=100, temp=1.0, row_temp=None,
            ids=P, ids_ld=1, m=1, logp=P, ent=P, lse=P, ws=P, wsb=1 << 30):
    return lib.zs_lmhead_logprobs(h, hidden, hld, norm, 1e-6, w, batch, E, V, temp, row_temp, ids,
                                  ids_ld, m, logp, ent, lse, ws, wsb, None)


@pytest.mark.parametrize("change", [
    dict(hidden=None), dict(norm=None), dict(w=None), dict(w=P + 8), dict(E=60), dict(E=56),
    dict(E=12296, hld=12296), dict(hld=63), dict(batch=-1), dict(V=0), dict(temp=float("nan")),
    dict(ids=None), dict(ids_ld=0), dict(m=257), dict(m=-1), dict(logp=None), dict(ent=P + 1),
    dict(row_temp=P + 1),
])
def test_lmhead_logprobs_refuses(lib, handle, change):
    assert _lmhead(lib, handle, **change) == BAD


def _embed(lib, h, table=P, td=BF16, tld=64, V=100, E=64, ids=P, n=3, out=P, od=F32, old=64):
    return lib.zs_embed(h, table, td, tld, V, E, ids, n, 1.0, out, od, old, None)


@pytest.mark.parametrize("change", [
    dict(table=None), dict(table=P + 1), dict(td=3), dict(od=-1), dict(tld=63), dict(old=63),
    dict(V=0), dict(E=0), dict(E=(1 << 20) + 1, tld=1 << 21, old=1 << 21), dict(ids=None),
    dict(ids=P + 1), dict(n=-1), dict(n=(1 << 30) + 1), dict(out=None), dict(out=P + 2),
    dict(tld=(1 << 40) + 1), dict(old=(1 << 40) + 1),
])
def test_embed_refuses(lib, handle, change):
    assert _embed(lib, handle, **change) == BAD


def _embed_backward(lib, h, g=P, gd=BF16, gld=64, ids=P, n=3, V=100, E=64, t=P, td=F32, tld=64,
                    acc=0, ws=P, wsb=1 << 30):
    return lib.zs_embed_backward(h, g, gd, gld, ids, n, 1.0, V, E, t, td, tld, acc, ws, wsb, None)


@pytest.mark.parametrize("change", [
    dict(g=None), dict(g=P + 1), dict(gd=3), dict(td=3), dict(gld=63), dict(tld=63), dict(V=0),
    dict(E=0), dict(ids=None), dict(ids=P + 2), dict(n=-1), dict(n=(1 << 30) + 1), dict(t=None),
    dict(t=P + 2), dict(ws=None), dict(ws=P + 128), dict(wsb=100), dict(tld=(1 << 40) + 1),
])
def test_embed_backward_refuses(lib, handle, change):
    assert _embed_backward(lib, handle, **change) == BAD


def test_empty_calls_do_nothing(lib, handle):
    assert _backward(lib, handle, batch=0) == 0
    assert _lmhead(lib, handle, batch=0) == 0
    assert _embed(lib, handle, n=0) == 0
    assert _embed_backward(lib, handle, n=0, acc=1, ws=None, wsb=0) == 0


def test_embed_backward_workspace(lib):
    out = C.c_int64()
    assert lib.zs_embed_backward_workspace(0, 8, C.byref(out)) == 0 and out.value >= 0
    last = 0
    for n in (1, 31, 32, 33, 1000, 100000):
        assert lib.zs_embed_backward_workspace(n, 64, C.byref(out)) == 0
        # the pairs, twice, and two partial rows per 32 positions
        assert out.value >= 16 * n + -(-n // 32) * 2 * 64 * 4
        assert out.value >= last
        last = out.value
    for n, e in ((-1, 8), ((1 << 30) + 1, 8), (4, 0), (4, (1 << 20) + 1)):
        assert lib.zs_embed_backward_workspace(n, e, C.byref(out)) == BAD
    assert lib.zs_embed_backward_workspace(4, 8, None) == BAD


# ---- the bounds of the top alternatives, from one key per thread ----

CODE_BITS = 12


def _order(v):
    """The kernels' 32-bit order of a float (NaN lowest)."""
    if np.isnan(v):
        return 0
    u = int(np.float32(v + 0.0).view(np.uint32))
    return u ^ 0xFFFFFFFF if u >> 31 else u | 0x80000000


def _key(v, i):
    return _order(v) << 32 | (~i & 0xFFFFFFFF)


def _bounds(x, k, head, N, nt, cl):
    """(rough, exact): the keys that zs_logprobs_kernel takes as lower bounds of the k best, on a
    row whose first `head` elements precede the first 16-byte boundary, with N elements per
    vector, nt threads and cl CTAs."""
    n = x.size
    head = min(head, n)
    nvec = (n - head) // N
    tail = n - head - nvec * N
    threads = []  # (rough key, exact key, up to its vector's last id)
    for r in range(cl):
        v0, v1 = nvec * r // cl, nvec * (r + 1) // cl
        for t in range(nt):
            units = [(t, 1)] if r == 0 and t < head else []
            units += [(head + v * N, N) for v in range(v0 + t, v1, nt)]
            if r == cl - 1 and t < tail:
                units.append((head + nvec * N + t, 1))
            if not units:
                continue
            best, (pos, span) = -np.inf, units[0]
            for p, s in units:
                m = x[p:p + s].max()
                if m > best:
                    best, pos, span = m, p, s
            code = (1 << CODE_BITS) - 1 - (r * nt + t)
            threads.append((_order(best) >> CODE_BITS << CODE_BITS | code, _key(best, pos + span - 1)))
    threads.sort(reverse=True)
    if len(threads) < k:
        return 0, 0
    sel = threads[:k]
    return (sel[-1][0] >> CODE_BITS << CODE_BITS) << 32, min(e for _, e in sel)


@pytest.mark.parametrize("kind", ["normal", "ties", "equal", "up", "down", "masked"])
@pytest.mark.parametrize("n,head,N,nt,cl,k", [(997, 3, 4, 32, 1, 5), (997, 0, 8, 16, 4, 16),
                                              (50, 1, 8, 32, 2, 20), (33, 5, 8, 16, 1, 16),
                                              (400, 2, 4, 64, 8, 33), (7, 0, 4, 8, 1, 5)])
def test_k_elements_reach_the_bounds(kind, n, head, N, nt, cl, k):
    """At least k elements have a key at or above either bound, so the k best do; and
    ties leave few above the exact one."""
    rng = np.random.default_rng(n + k)
    for _ in range(5):
        x = {"normal": rng.normal(size=n), "ties": np.round(rng.normal(size=n) * 2),
             "equal": np.zeros(n), "up": np.arange(n) * 1.0, "down": -np.arange(n) * 1.0,
             "masked": np.where(rng.random(n) < 0.97, -np.inf, rng.normal(size=n))}[kind]
        x = x.astype(np.float32)
        keys = [_key(v, i) for i, v in enumerate(x)]
        rough, exact = _bounds(x, k, head, N, nt, cl)
        assert sum(q >= rough for q in keys) >= k
        assert sum(q >= exact for q in keys) >= k
        if kind == "equal" and exact:
            assert sum(q >= exact for q in keys) <= nt * cl * N + head
