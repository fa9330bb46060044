"""Sampler.embed and Sampler.embed_backward against plain torch.

embed is one f32 product rounded once, so it has to agree bit for bit.  The gradient of an
id with c rows is a sum of c f32 terms (c - 1 roundings of partial sums, each at most half
a step u = 2^-24 of the sum of magnitudes), scaled (u) and rounded to the table's type."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def ids_of(n, V, seed=0, outside=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.exp(torch.rand(n, generator=g) * math.log(V + 1.0)).long().sub(1).clamp_(0, V - 1)
    if outside and n > 2:
        ids[n // 2] = -1
        ids[n // 3] = V
        ids[0] = -2 ** 31
    return ids.to(torch.int32).cuda()


def plain(table, ids, scale, dtype):
    V = table.shape[0]
    ok = (ids >= 0) & (ids < V)
    rows = table[ids.long().clamp(0, V - 1)].float() * scale
    return torch.where(ok[..., None], rows, 0.0).to(dtype)


@pytest.mark.parametrize("td", TYPES)
@pytest.mark.parametrize("od", TYPES)
@pytest.mark.parametrize("n,V,E", [(1, 1, 1), (3, 5, 7), (64, 1000, 896), (5, 300, 260), (33, 100, 1028),
                                   (5000, 777, 96), (20000, 4000, 8)])
def test_embed(sampler, td, od, n, V, E):
    table = torch.randn(V, E, device="cuda").to(td)
    ids = ids_of(n, V)
    for scale in (1.0, 0.37):
        got = sampler.embed(table, ids, scale=scale, out_dtype=od)
        assert got.dtype == od and torch.equal(got, plain(table, ids, scale, od))


def test_embed_strides_shapes_and_streams(sampler):
    buf = torch.randn(50, 72, device="cuda").to(BF16)
    ids = ids_of(12, 50).reshape(3, 4)
    for table in (buf[:, :64], buf[:, 1:65], buf[:, 3:67], buf[:, :61]):
        E = table.shape[1]
        want = plain(table, ids, 2.0, F32)
        assert torch.equal(sampler.embed(table, ids, 2.0, out_dtype=F32), want)
        out = torch.full((12, E + 3), 7.0, device="cuda")
        sampler.embed(table, ids, 2.0, out=out[:, 1:E + 1])
        assert torch.equal(out[:, 1:E + 1], want.reshape(12, E))
        assert (out[:, 0] == 7).all() and (out[:, E + 1:] == 7).all()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = sampler.embed(table, ids, 2.0, out_dtype=F32, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
    assert sampler.embed(buf, ids[:0].reshape(0)).shape == (0, 72)


def test_embed_of_a_decode_step(sampler):
    """The ids of a decode step, one sequence stopped, through the tied lm_head weights."""
    from zeninfer_b200 import SamplingParams, states_to_tensor
    import numpy as np
    logits = torch.randn(4, 1000, device="cuda") * 3
    w = torch.randn(1000, 64, device="cuda").to(BF16)
    done = torch.tensor([0, 1, 0, 0], dtype=torch.int32, device="cuda")
    st = states_to_tensor(np.arange(1, 5, dtype=np.uint64), logits.device)
    ids = sampler.decode_step(logits, SamplingParams(temp=0.7, top_k=40), st, done, eos=999)
    r = sampler.logprobs(logits, ids, temp=0.7, top=5)
    x = sampler.embed(w, ids, scale=8.0, out_dtype=F32)
    nxt = sampler.lmhead_logprobs(x, torch.ones(64, device="cuda"), w, ids)
    assert int(ids[1]) == -1 and float(r.logp[1]) == 0.0 and float(nxt.logp[1]) == 0.0
    assert not x[1].any()
    keep = [0, 2, 3]
    assert torch.equal(x[keep], w[ids[keep].long()].float() * 8.0)
    assert (r.logp[keep] < 0).all() and (nxt.logp[keep] <= 0).all()


def exact_grad(grad, ids, V, scale):
    """(gradient, count of rows, sum of magnitudes) per table row in 64 bits."""
    ok = (ids >= 0) & (ids < V)
    at = ids.long()[ok]
    E = grad.shape[1]
    z = torch.zeros(V, E, dtype=torch.float64, device="cuda")
    want = z.index_add(0, at, grad[ok].double()) * scale
    mag = z.index_add(0, at, grad[ok].double().abs()) * abs(scale)
    cnt = torch.zeros(V, dtype=torch.float64, device="cuda").index_add(
        0, at, torch.ones(at.numel(), dtype=torch.float64, device="cuda"))
    return want, cnt[:, None], mag


def check_grad(got, grad, ids, V, scale, base=None):
    want, cnt, mag = exact_grad(grad, ids, V, scale)
    f = torch.finfo(got.dtype)
    if base is not None:
        want, mag = want + base.double(), mag + base.double().abs()
    tol = (cnt + 2) * U * mag * 1.01 + want.abs() * f.eps / 2 * 1.01 + f.tiny * f.eps / 2
    off = (got.double() - want).abs()
    assert not (off > tol).any(), f"{int((off > tol).sum())} off, worst {float((off - tol).max())}"
    untouched = (cnt == 0)[:, 0]
    assert torch.equal(got[untouched], torch.zeros_like(got[untouched]) if base is None
                       else base[untouched])


@pytest.mark.parametrize("gd", TYPES)
@pytest.mark.parametrize("td", TYPES)
@pytest.mark.parametrize("n,V,E", [(1, 1, 1), (2, 600, 16), (31, 40, 7), (33, 5, 64), (1000, 3000, 100),
                                   (9000, 151936, 8), (3000, 511, 264), (2500, 512, 1032)])
def test_embed_backward(sampler, gd, td, n, V, E):
    g = torch.Generator(device="cuda").manual_seed(n)
    grad = torch.randn(n, E, generator=g, device="cuda").to(gd)
    ids = ids_of(n, V, seed=n)
    got = sampler.embed_backward(grad, ids, V, scale=0.5, dtype=td)
    assert got.dtype == td and got.shape == (V, E)
    check_grad(got, grad, ids, V, 0.5)
    assert torch.equal(got, sampler.embed_backward(grad, ids, V, scale=0.5, dtype=td))
    base = torch.randn(V, E, generator=g, device="cuda").to(td)
    acc = base.clone()
    sampler.embed_backward(grad, ids, V, scale=0.5, out=acc, accumulate=True)
    check_grad(acc, grad, ids, V, 0.5, base)


@pytest.mark.parametrize("kind", ["one", "two", "all_different", "descending", "outside", "borders"])
@pytest.mark.parametrize("n", [1, 32, 64, 65, 4097, 70000])
def test_embed_backward_runs(sampler, kind, n):
    """Small whole numbers: every f32 sum is exact, so the order cannot matter and the
    result has to be equal."""
    V, E = 1 << 17, 16
    i = torch.arange(n)
    ids = {"one": torch.full((n,), 77), "two": 5 + 1000 * (i % 2), "all_different": (i * 7919) % V,
           "descending": V - 1 - i, "outside": torch.where(i % 3 == 0, i % 50, V + i),
           "borders": (i + 16) // 32}[kind].to(torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    grad = torch.randint(-3, 4, (n, E), generator=g, device="cuda").float()
    want = exact_grad(grad, ids, V, 1.0)[0].float()
    assert torch.equal(sampler.embed_backward(grad, ids, V), want)


@pytest.mark.parametrize("td", TYPES)
@pytest.mark.parametrize("n", [0, 3, 1024, 1025])
@pytest.mark.parametrize("V,E", [(5000, 33), (4999, 32), (100, 2049), (37, 9000), (9, 1), (4001, 6)])
def test_embed_backward_zeroes_the_rest(sampler, td, n, V, E):
    """Rows that no token names are zero whatever was there, in tables whose rows do and do
    not start at 16-byte boundaries, contiguous or not; nothing else is touched."""
    ids = ids_of(n, V, seed=5)
    grad = torch.ones(n, E, device="cuda")
    want = exact_grad(grad, ids, V, 1.0)[0].to(td)  # whole numbers: exact up to the rounding
    for off, ld in ((0, E), (1, E), (0, E + 1), (0, E + 8 - E % 8)):
        buf = torch.full((off + V * ld + 64,), 5.0, device="cuda", dtype=td)
        view = torch.as_strided(buf, (V, E), (ld, 1), off)
        sampler.embed_backward(grad, ids, V, out=view)
        assert torch.equal(view, want)
        view.fill_(5.0)
        assert (buf == 5.0).all()  # nothing else was touched (an id may occur five times)


def test_embed_backward_strides_streams_and_graphs(sampler):
    n, V, E = 700, 90, 40
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn(n, E + 8, generator=g, device="cuda").to(BF16)
    ids = ids_of(n, V, seed=4)
    for off in (0, 1, 8):
        grad = wide[:, off:off + E]
        ref = sampler.embed_backward(grad, ids, V, dtype=F32)
        check_grad(ref, grad, ids, V, 1.0)
        out = torch.full((V, E + 4), 3.0, device="cuda")
        for view in (out[:, :E], out[:, 3:3 + E]):
            out.fill_(3.0)
            sampler.embed_backward(grad, ids, V, out=view)
            assert torch.equal(view, ref)
            assert int((out == 3.0).sum()) >= V * 4
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        a = sampler.embed_backward(grad, ids, V, dtype=F32, stream=side)
        b = sampler.embed_backward(grad, ids, V, dtype=F32)
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs = [], []
        for _ in range(2):  # two graphs, each with a workspace of its own pool
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(sampler.embed_backward(grad, ids, V, dtype=F32))
            graphs.append(graph)
        for graph in graphs + graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in (a, b, *outs):
            assert torch.equal(got, ref)


def test_offsets_past_32_bits(sampler):
    V, E = 2_800_000, 800  # 2.24 G elements
    table = torch.zeros(V, E, dtype=torch.float16, device="cuda")
    ids = torch.tensor([V - 1, 0, V - 2, 5, V - 1], dtype=torch.int32, device="cuda")
    grad = torch.randint(-4, 5, (5, E), device="cuda").to(torch.float16)
    for n in (5, 2000):  # above 1024 tokens, and above 2^19 ids, the sorted way
        i2, g2 = ids.repeat(n // 5), grad.repeat(n // 5, 1)
        table.fill_(1.0)
        sampler.embed_backward(g2, i2, V, out=table)
        assert torch.equal(table[V - 1], (grad[0] + grad[4]) * (n // 5))
        assert torch.equal(table[V - 2], grad[2] * (n // 5)) and torch.equal(table[5], grad[3] * (n // 5))
        assert not table[6:V - 2].any() and not table[1:5].any()
    assert torch.equal(sampler.embed(table, ids), table[ids.long()])
    wide = torch.as_strided(table, (2, E), (V * E - E, 1))
    assert torch.equal(sampler.embed(table[:3], torch.zeros(2, dtype=torch.int32, device="cuda"), 1.0,
                                     out=wide), table[[0, V - 1]])


def test_embed_backward_on_two_streams_at_once(sampler):
    n, V, E = 9000, 4000, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    grads = [torch.randn(n, E, generator=g, device="cuda") for _ in range(2)]
    ids = [ids_of(n, V, seed=40 + i) for i in range(2)]
    want = [sampler.embed_backward(grads[i], ids[i], V) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(8):
        for i, st in enumerate(streams):
            got.append((i, sampler.embed_backward(grads[i], ids[i], V, stream=st)))
    torch.cuda.synchronize()
    for i, t in got:
        assert torch.equal(t, want[i])


def test_embed_backward_against_differences(sampler):
    """The loss sum(embed(table) * grad) is linear in the table: its difference quotient is
    the gradient (64-bit sums; f32 roundings of a few terms of order 1)."""
    V, E, n = 6, 4, 10
    ids = torch.tensor([0, 1, 1, 5, -1, 5, 5, 2, 6, 0], dtype=torch.int32, device="cuda")
    grad = torch.randn(n, E, device="cuda")
    got = sampler.embed_backward(grad, ids, V, scale=1.5)
    table = torch.zeros(V, E, device="cuda")
    for v in range(V):
        for e in range(E):
            table.zero_()
            table[v, e] = 1.0
            loss = (sampler.embed(table, ids, 1.5).double() * grad.double()).sum()
            assert abs(float(loss) - float(got[v, e])) < 1e-5


def test_empty_calls(sampler):
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    z = sampler.embed_backward(torch.empty(0, 24, device="cuda"), none, 7)
    assert z.shape == (7, 24) and not z.any()
    base = torch.ones(7, 24, device="cuda")
    sampler.embed_backward(torch.empty(0, 24, device="cuda"), none, 7, out=base, accumulate=True)
    assert (base == 1).all()


def test_refusals(sampler):
    table = torch.randn(10, 16, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    grad = torch.randn(4, 16, device="cuda")
    for a, kw in (((table.double(), ids), {}), ((table.cpu(), ids), {}), ((table[0], ids), {}),
                  ((table.t(), ids), {}), ((table, ids.long()), {}), ((table, ids.cpu()), {}),
                  ((table, torch.zeros(8, dtype=torch.int32, device="cuda")[::2]), {}),
                  ((table, ids), dict(out_dtype=torch.float64)),
                  ((table, ids), dict(out=torch.empty(4, 15, device="cuda"))),
                  ((table, ids), dict(out=torch.empty(4, 16, device="cuda"), out_dtype=F16))):
        with pytest.raises(ValueError):
            sampler.embed(*a, **kw)
    for a, kw in (((grad, ids[:3], 10), {}), ((grad.double(), ids, 10), {}), ((grad, ids.long(), 10), {}),
                  ((grad, ids, 10), dict(accumulate=True)), ((grad, ids, 10), dict(dtype=torch.int32)),
                  ((grad, ids, 10), dict(out=torch.empty(9, 16, device="cuda"))),
                  ((grad, ids, 10), dict(out=torch.empty(10, 16, device="cuda"), dtype=BF16)),
                  ((grad[:, :1].expand(4, 16), ids, 10), {})):
        with pytest.raises(ValueError):
            sampler.embed_backward(*a, **kw)
    from zeninfer_b200._native import SamplerError
    with pytest.raises(SamplerError):
        sampler.embed_backward(grad, ids, 0, out=torch.empty(0, 16, device="cuda"))
