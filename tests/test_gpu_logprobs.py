"""Sampler.logprobs, its gradient and Sampler.lmhead_logprobs against 64-bit torch.

Tolerances, with u = 2^-24 (half a step of f32), d = (x - max) / temp and p = softmax:
an exponent d carries three f32 roundings (the difference, inv_temp * log2 e and their
product), so e^d is off by at most 3 |d| u, plus 4 u for the exponential itself; a sum
over n terms in f32 with at most n / 256 + 64 terms in one chain, each possibly rescaled
(5 u), adds DEPTH(n) u.  Hence
    lse      (3 E|d| + 4 + DEPTH) u, and half a step of the result
    entropy  that + (3 E d^2 + (10 + DEPTH) E|d|) u + E|d| times lse's, and half a step
    log p    lse's and half a step
    gradient of one element: (3 |d| + 10) u of its terms' magnitudes, and half a step
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def depth(n):
    return 6 * (math.ceil(n / 256) + 64)


def inv_temp(temp):
    t = np.float32(temp)
    return 1.0 if t <= 0 else float(np.float32(1.0) / t)


def exact(x, it):
    """(lse, entropy, log p, tolerances of lse and entropy) of rows x in 64 bits; it: [B]."""
    z = x.double() * it[:, None]
    m = z.max(1).values
    dead = torch.isneginf(m)
    # from the maximum: next to f32's lowest value, z - lse would lose log s even in 64 bits
    t = z - torch.where(dead, 0.0, m)[:, None]
    log_s = torch.logsumexp(t, 1)
    lse = m + log_s
    logp = torch.where(dead[:, None], -math.inf, t - torch.where(dead, 0.0, log_s)[:, None])
    p = torch.exp(logp)
    h = -(p * torch.where(p > 0, logp, 0.0)).sum(1)
    d = torch.where(p > 0, z - z.max(1, keepdim=True).values, 0.0)
    e1, e2 = (p * d.abs()).sum(1), (p * d * d).sum(1)
    n = x.shape[1]
    t_sum = (3 * e1 + 4 + depth(n)) * U
    t_lse = t_sum + lse.abs().nan_to_num(posinf=0.0) * U
    t_h = t_sum * (1 + e1) + (3 * e2 + (10 + depth(n)) * e1) * U + h.abs() * U
    return lse, h, logp, t_sum, t_lse, t_h


def close(got, want, tol, what):
    got, want = got.double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} values off, worst "
                           f"{float((got - want).abs()[bad].nan_to_num().max())}")


def order(x, k):
    """The k best ids of every row, value descending (NaN last), then id ascending."""
    v = x.float().cpu().numpy()
    out = np.empty((v.shape[0], k), np.int64)
    for r in range(v.shape[0]):
        key = np.where(np.isnan(v[r]), -np.inf, v[r])
        out[r] = np.lexsort((np.arange(v.shape[1]), -key, np.isnan(v[r])))[:k]
    return torch.from_numpy(out)


def check(s, x, ids, temp=1.0, top=0, **kw):
    B, V = x.shape
    r = s.logprobs(x, ids, temp=temp, top=top, **kw)
    torch.cuda.synchronize()
    it = torch.tensor([inv_temp(t) for t in (temp.tolist() if isinstance(temp, torch.Tensor)
                                             else [temp] * B)], dtype=torch.float64, device=x.device)
    lse, h, logp, t_sum, t_lse, t_h = exact(x, it)
    close(r.lse, lse, t_lse, "lse")
    close(r.entropy, h, t_h, "entropy")
    if ids is not None:
        i2 = ids.long().reshape(B, -1)
        inside = (i2 >= 0) & (i2 < V)
        want = torch.where(inside, torch.gather(logp, 1, i2.clamp(0, V - 1)), 0.0)
        tol = t_sum[:, None] + want.abs().nan_to_num(posinf=0.0) * U
        close(r.logp.reshape(B, -1), want, tol, "logp")
        assert r.logp.shape == ids.shape
    if top > 0:
        k = min(top, V)
        want_ids = order(x, k).to(x.device)
        assert torch.equal(r.top_ids.long(), want_ids)
        want = torch.gather(logp, 1, want_ids)
        close(r.top_logp, want, t_sum[:, None] + want.abs().nan_to_num(posinf=0.0) * U, "top_logp")
    return r


def rand(B, V, dtype, seed=0, scale=2.5, off=0, ld=None):
    """[B, V] logits that start `off` elements into their buffer, rows `ld` apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or V
    buf = (torch.randn(off + B * ld, generator=g, device="cuda") * scale).to(dtype)
    return torch.as_strided(buf, (B, V), (ld, 1), off)


def some_ids(B, V, m, seed=1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (B, m), generator=g, dtype=torch.int32)
    ids[0, 0] = -1
    if m > 1:
        ids[-1, 1] = ids[-1, 0]
        ids[B // 2, m - 1] = V
    return ids.cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,V,off,ld,m,top", [
    (1, 1, 0, None, 1, 1), (2, 2, 1, 3, 1, 5), (3, 5, 0, None, 2, 3), (1, 100, 3, None, 4, 64),
    (7, 1000, 0, None, 1, 128), (5, 4099, 1, None, 3, 20), (2, 32768, 0, 32776, 1, 5),
    (1, 50001, 0, None, 1, 7), (40, 5003, 5, 5010, 1, 0), (1300, 2001, 0, None, 1, 4),
    (9, 65536, 0, None, 2, 128), (10, 40001, 2, 40003, 1, 33),
])
def test_logprobs(sampler, dtype, B, V, off, ld, m, top):
    check(sampler, rand(B, V, dtype, off=off, ld=ld), some_ids(B, V, m), 0.7, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [129, 520, 1030, 3000, 8200])
def test_many_alternatives_of_short_rows(sampler, dtype, V):
    """Fewer vectors than, or about as many as, threads and alternatives."""
    for off in (0, 3):
        check(sampler, rand(3, V, dtype, seed=V, off=off), None, 1.0, 128)


def test_rows_longer_than_the_kept_segments(sampler):
    """Slices of more than 2 MB, whose segments' maxima are not kept."""
    check(sampler, rand(1, 5_000_003, torch.float32, seed=1), some_ids(1, 5_000_003, 1), 1.0, 3)
    x = rand(300, 700_001, torch.bfloat16, seed=2)
    r = sampler.logprobs(x, top=2)
    assert torch.equal(r.top_ids[::60].long(), order(x[::60], 2).to(x.device))
    y = rand(300, 1_100_001, torch.bfloat16, seed=3)
    r = sampler.logprobs(y, top=2)
    assert torch.equal(r.top_ids[::100].long(), order(y[::100], 2).to(x.device))


def test_logprobs_qwen_vocabulary(sampler):
    for B, dtype in ((1, torch.float32), (3, torch.bfloat16), (64, torch.float32)):
        check(sampler, rand(B, 151936, dtype, seed=B), some_ids(B, 151936, 1), 0.7, 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [1, 30])
def test_ties_take_the_lowest_id(sampler, dtype, B):
    V = 20003
    x = rand(B, V, dtype, seed=3)
    check(sampler, (x.float().round() * 1.0).to(dtype), None, 1.0, 100)
    check(sampler, torch.zeros(B, V, dtype=dtype, device="cuda"), None, 1.0, 128)
    both = torch.zeros(B, V, dtype=dtype, device="cuda")
    both[:, ::2] = -0.0  # -0 and +0 are one value
    check(sampler, both, None, 1.0, 9)


@pytest.mark.parametrize("B", [1, 200])
def test_sorted_rows(sampler, B):
    x = torch.arange(30011, device="cuda", dtype=torch.float32).repeat(B, 1) * 1e-3
    check(sampler, x, None, 1.0, 50)
    check(sampler, -x, None, 1.0, 50)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [1, 9, 200])
@pytest.mark.parametrize("top", [0, 2])
def test_rows_that_outgrow_their_beginning(sampler, dtype, B, top):
    """Values that rise by far more than the exponential's range, a single peak at the
    end, a fall from a first peak, and a first part without any token."""
    V = 40013
    x = rand(B, V, dtype, seed=21)
    ramp = torch.linspace(-300, 300, V, device="cuda")
    rows = [x + ramp, x - ramp, x.clone(), x.clone(), x.clone()]
    rows[2][:, V - 1] = 60000.0
    rows[3][:, 0] = 500.0
    rows[4][:, :V - 900] = -math.inf
    for y in rows:
        check(sampler, y.to(dtype), some_ids(B, V, 1), 1.0, top)
        check(sampler, y.to(dtype), some_ids(B, V, 1), 0.1, top)
        check(sampler, y.to(dtype), some_ids(B, V, 1), 30.0, top)


def test_offsets_past_32_bits(sampler):
    V, ld = 1500, (1 << 31) + 8
    buf = torch.empty(ld + V, dtype=torch.float16, device="cuda")
    x = torch.as_strided(buf, (2, V), (ld, 1), 0)
    x.copy_(rand(2, V, torch.float16, seed=22))
    ids = some_ids(2, V, 1)
    r = check(sampler, x, ids, 1.0, 5)
    gl = torch.ones(2, 1, device="cuda")
    want = sampler.logprobs_backward(x.contiguous(), r.rows, ids, gl)
    sampler.logprobs_backward(x, r.rows, ids, gl, out=x)
    assert torch.equal(x, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [4, 150])
def test_masked_rows(sampler, dtype, B):
    V = 12001
    g = torch.Generator(device="cuda").manual_seed(5)
    x = rand(B, V, dtype, seed=5)
    x.masked_fill_(torch.rand(B, V, generator=g, device="cuda") < 0.999, -math.inf)
    x[1] = -math.inf                      # nothing left
    x[2] = -math.inf
    x[2, V - 1] = 1.0                     # one token left
    r = check(sampler, x, some_ids(B, V, 2), 1.3, 40)
    assert float(r.entropy[2]) == 0.0 and float(r.lse[1]) == -math.inf
    low = torch.finfo(dtype).min          # masks of the type's lowest value
    y = torch.where(torch.isinf(x), low, x)
    check(sampler, y, some_ids(B, V, 2), 1.0, 10)
    y[0] = low                            # ... in every place: an even row
    r = check(sampler, y, some_ids(B, V, 1), 1.0, 5)
    assert abs(float(r.entropy[0]) - math.log(V)) < 1e-5


@pytest.mark.parametrize("B", [3, 150])
def test_nan_and_inf_rows(sampler, B):
    V = 9001
    x = rand(B, V, torch.float32, seed=8)
    x[0, 17] = math.nan
    x[1, 0] = math.inf
    x[2] = math.nan
    r = sampler.logprobs(x, some_ids(B, V, 1).clamp_(min=0), top=6)
    for row in (0, 1, 2):
        assert r.lse[row].isnan() and r.entropy[row].isnan() and r.logp[row].isnan().all()
    assert torch.equal(r.top_ids.cpu().long(), order(x, 6))
    if B > 3:
        check(sampler, x[3:], None, 1.0, 6)
    # fewer numbers than alternatives, the rest NaN
    y = torch.full((B, V), math.nan, device="cuda")
    y[:, 4000] = 1.0
    y[:, 4001] = -math.inf
    y[:, 8999] = 1.0
    r = sampler.logprobs(y, top=5)
    assert r.top_ids[B - 1].tolist() == [4000, 8999, 4001, 0, 1]


def test_row_temperatures(sampler):
    B, V = 33, 7001
    temp = torch.linspace(0.2, 3.0, B, device="cuda")
    temp[4] = 0.0    # greedy rows count as 1
    temp[5] = -1.0
    check(sampler, rand(B, V, torch.float32, seed=4), some_ids(B, V, 1), temp, 3)


def test_log_z_of_sample_agrees(sampler):
    from zeninfer_b200 import SamplingParams, states_to_tensor
    x = rand(6, 151936, torch.float32, seed=6)
    st = states_to_tensor(np.arange(1, 7, dtype=np.uint64), x.device)
    info = sampler.sample(x, SamplingParams(temp=0.7, top_k=40), st, row_info=True,
                          want_log_z=True).row_info
    r = sampler.logprobs(x, temp=0.7)
    want = info["log_z"] + info["max_logit"].astype(np.float64) * inv_temp(0.7)
    assert np.allclose(r.lse.cpu().numpy(), want, rtol=0, atol=2e-5)


# ---- gradient ----

def exact_grad(x, rows, ids, gl, gh, gz):
    """(gradient, tolerance before the last rounding) from the forward pass's rows."""
    rows = rows.double()
    m, s, h, it = rows[:, 0:1], rows[:, 1:2], rows[:, 2:3], rows[:, 3:4]
    dead = s == 0
    d = torch.where(dead, 0.0, (x.double() - torch.where(dead, 0.0, m)) * it)
    p = torch.where(dead, 0.0, torch.exp(d) / torch.where(dead, 1.0, s))
    logp = torch.where(p > 0, d - torch.log(torch.where(dead, 1.0, s)), 0.0)
    B, V = x.shape
    gh = torch.zeros(B, 1, dtype=torch.float64, device=x.device) if gh is None else gh.double()[:, None]
    gz = torch.zeros(B, 1, dtype=torch.float64, device=x.device) if gz is None else gz.double()[:, None]
    delta = torch.zeros(B, V, dtype=torch.float64, device=x.device)
    mag = delta.clone()
    G = torch.zeros(B, 1, dtype=torch.float64, device=x.device)
    GA = G.clone()
    if ids is not None:
        i2, g2 = ids.long().reshape(B, -1), gl.double().reshape(B, -1)
        ok = (i2 >= 0) & (i2 < V) & ~dead
        inside = (i2 >= 0) & (i2 < V)
        G = (g2 * inside).sum(1, keepdim=True)
        GA = (g2.abs() * inside).sum(1, keepdim=True)
        delta.scatter_add_(1, i2.clamp(0, V - 1), g2 * ok)
        mag.scatter_add_(1, i2.clamp(0, V - 1), g2.abs() * ok)
    want = it * (delta + p * (gz - G - gh * h - gh * logp))
    size = p * (gz.abs() + GA * 20 + gh.abs() * (h.abs() + torch.log(torch.where(dead, 1.0, s)).abs() * 2
                                                 + d.abs().nan_to_num(posinf=0.0)))
    tol = it * (size * (3 * d.abs().nan_to_num(posinf=0.0) + 10) + 20 * mag) * U
    return want, tol


def check_grad(got, x, rows, ids, gl, gh, gz):
    want, tol = exact_grad(x, rows, ids, gl, gh, gz)
    f = torch.finfo(x.dtype)
    # half a step of the result (eps / 2, or of the smallest subnormal), and values whose
    # p is below f32's normal range, which the exponential flushes to 0
    tol = tol * 1.01 + want.abs() * f.eps / 2 + f.tiny * f.eps / 2 + 2.0 ** -125
    close(got, want, tol, "gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,V,off,ld,m", [
    (1, 1, 0, None, 1), (2, 3, 1, 5, 2), (3, 4099, 0, None, 1), (5, 8192, 0, 8200, 4),
    (4, 20011, 3, None, 256), (70, 5003, 1, 5004, 1),
])
def test_gradient(sampler, dtype, B, V, off, ld, m):
    x = rand(B, V, dtype, seed=7, off=off, ld=ld)
    ids = some_ids(B, V, m)
    g = torch.Generator(device="cuda").manual_seed(9)
    gl = torch.randn(B, m, generator=g, device="cuda")
    gh, gz = (torch.randn(B, generator=g, device="cuda") for _ in range(2))
    r = sampler.logprobs(x, ids, temp=0.8)
    for a in ((ids, gl, gh, gz), (ids, gl, None, None), (None, None, gh, None),
              (None, None, None, gz)):
        got = sampler.logprobs_backward(x, r.rows, a[0], grad_logp=a[1], grad_entropy=a[2],
                                        grad_lse=a[3])
        assert got.dtype == dtype and got.shape == x.shape
        check_grad(got, x, r.rows, *a)
    # into a buffer whose rows start elsewhere, and in place
    out = rand(B, V, dtype, seed=2, off=off + 1, ld=(ld or V) + 3)
    guard = torch.as_strided(out, (B, 3), ((ld or V) + 3, 1), off + 1 + V).clone()
    sampler.logprobs_backward(x, r.rows, ids, gl, gh, gz, out=out)
    check_grad(out, x, r.rows, ids, gl, gh, gz)
    left = torch.as_strided(out, (B, 3), ((ld or V) + 3, 1), off + 1 + V)
    assert torch.equal(left[:-1], guard[:-1])
    same = x.clone() if ld is None else x
    before = same.clone()
    sampler.logprobs_backward(same, r.rows, ids, gl, gh, gz, out=same)
    check_grad(same, before, r.rows, ids, gl, gh, gz)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_masked_rows(sampler, dtype):
    B, V = 6, 9001
    x = rand(B, V, dtype, seed=11)
    x[:, ::3] = -math.inf
    x[1] = -math.inf
    x[2] = torch.finfo(dtype).min
    x[3, 1:] = torch.finfo(dtype).min
    ids = some_ids(B, V, 2)
    ids[1] = 7
    gl = torch.ones(B, 2, device="cuda")
    gh = torch.full((B,), 0.5, device="cuda")
    r = sampler.logprobs(x, ids)
    got = sampler.logprobs_backward(x, r.rows, ids, gl, gh, gh)
    assert not got.isnan().any()
    assert not got[1].any()
    assert not got[0, ::3][~torch.isin(torch.arange(0, V, 3, device="cuda"), ids[0])].any()
    check_grad(got, x, r.rows, ids, gl, gh, gh)
    x[4, 5] = math.nan
    r = sampler.logprobs(x, ids)
    assert sampler.logprobs_backward(x, r.rows, ids, gl)[4].isnan().all()


def test_gradient_against_differences(sampler):
    """Central differences of the 64-bit loss, step h: the gradient's error is h^2 / 6 times
    the third derivative (below 10 here), that is below 2e-6 at h = 1e-3, plus f32 roundings
    (values of order 1: below 1e-5)."""
    B, V, it = 3, 41, inv_temp(0.7)
    x = rand(B, V, torch.float32, seed=12, scale=1.0)
    ids = torch.tensor([[3, 3], [40, -1], [0, 7]], dtype=torch.int32, device="cuda")
    gl = torch.tensor([[0.5, -0.25], [1.0, 9.0], [-0.75, 0.3]], device="cuda")
    gh = torch.tensor([0.2, -0.4, 0.0], device="cuda")
    gz = torch.tensor([0.0, 0.1, -0.3], device="cuda")

    def loss(z):
        z = z * it
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        h = -(lp.exp() * lp).sum(1)
        got = torch.gather(lp, 1, ids.clamp(min=0).long()) * (ids >= 0)
        return float((got * gl).sum() + (h * gh).sum() + (torch.logsumexp(z, 1) * gz).sum())

    r = sampler.logprobs(x, ids, temp=0.7)
    got = sampler.logprobs_backward(x, r.rows, ids, gl, gh, gz).double()
    for b in range(B):
        for v in range(V):
            step = torch.zeros(B, V, dtype=torch.float64, device="cuda")
            step[b, v] = 1e-3
            want = (loss(x.double() + step) - loss(x.double() - step)) / 2e-3
            assert abs(float(got[b, v]) - want) < 1.2e-5


# ---- streams, graphs, refusals ----

def test_streams_graphs_and_repeats(sampler):
    B, V = 21, 30001
    x = rand(B, V, torch.bfloat16, seed=13)
    ids = some_ids(B, V, 2)
    gl = torch.ones(B, 2, device="cuda")
    ref = sampler.logprobs(x, ids, top=9)
    ref_g = sampler.logprobs_backward(x, ref.rows, ids, gl)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = []
    for stream in (side, None, side):
        r = sampler.logprobs(x, ids, top=9, stream=stream)
        outs.append((r, sampler.logprobs_backward(x, r.rows, ids, gl, stream=stream)))
        if stream is not None:
            torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = sampler.logprobs(x, ids, top=9)
        g = sampler.logprobs_backward(x, r.rows, ids, gl)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    outs.append((r, g))
    for r, g in outs:
        for name in ("logp", "entropy", "lse", "top_ids", "top_logp", "rows"):
            assert torch.equal(getattr(r, name), getattr(ref, name)), name
        assert torch.equal(g, ref_g)


def test_two_streams_at_once(sampler):
    """Calls that overlap on the GPU share nothing."""
    B, V = 300, 30011
    xs = [rand(B, V, torch.float32, seed=30 + i) for i in range(2)]
    ids = some_ids(B, V, 1)
    gl = torch.ones(B, 1, device="cuda")
    hidden, norm, w = lm_inputs(64, 5000, 256, seed=9)
    want = [sampler.logprobs(x, ids, top=20) for x in xs]
    want_g = [sampler.logprobs_backward(x, r.rows, ids, gl) for x, r in zip(xs, want)]
    want_l = [sampler.lmhead_logprobs(hidden * (i + 1), norm, w, temp=1.0 + i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    hs = [hidden * (i + 1) for i in range(2)]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, st in enumerate(streams):
            r = sampler.logprobs(xs[i], ids, top=20, stream=st)
            g = sampler.logprobs_backward(xs[i], r.rows, ids, gl, stream=st)
            got[i].append((r, g, sampler.lmhead_logprobs(hs[i], norm, w, temp=1.0 + i, stream=st)))
    torch.cuda.synchronize()
    for i in range(2):
        for r, g, lm in got[i]:
            assert torch.equal(r.logp, want[i].logp) and torch.equal(r.top_ids, want[i].top_ids)
            assert torch.equal(g, want_g[i])
            assert torch.equal(lm.lse, want_l[i].lse) and torch.equal(lm.entropy, want_l[i].entropy)


def test_empty_and_no_ids(sampler):
    r = sampler.logprobs(torch.empty(0, 100, device="cuda"), top=3)
    assert r.entropy.shape == (0,) and r.top_ids.shape == (0, 3) and r.logp is None
    x = rand(2, 50, torch.float32)
    assert sampler.logprobs(x, torch.empty(2, 0, dtype=torch.int32, device="cuda")).logp.shape == (2, 0)
    assert sampler.logprobs(x[0]).lse.shape == (1,)


def test_refusals(sampler):
    from zeninfer_b200._native import SamplerError
    x = rand(4, 100, torch.float32)
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    r = sampler.logprobs(x, ids)
    for bad in (dict(ids=ids.long()), dict(ids=ids[:2]), dict(ids=ids.cpu()),
                dict(temp=torch.ones(3, device="cuda")), dict(temp=torch.ones(4))):
        with pytest.raises(ValueError):
            sampler.logprobs(x, **{"ids": ids, **bad})
    for y in (x.double(), x.cpu(), x.t(), x[0].expand(3, 100)):
        with pytest.raises(ValueError):
            sampler.logprobs(y)
    with pytest.raises(SamplerError):
        sampler.logprobs(x, ids, temp=math.nan)
    for y, top in ((x, -1), (rand(1, 500, torch.float32), 129)):
        with pytest.raises(ValueError):
            sampler.logprobs(y, top=top)
    with pytest.raises(SamplerError):
        sampler.logprobs(x, torch.zeros(4, 257, dtype=torch.int32, device="cuda"))
    g = torch.ones(4, device="cuda")
    for bad in (dict(grad_logp=g), dict(ids=ids, grad_logp=torch.ones(4, 2, device="cuda")),
                dict(grad_entropy=g[:3]), dict(grad_lse=g.double()), dict(out=torch.empty(4, 99, device="cuda")),
                dict(out=torch.empty(4, 100, device="cuda", dtype=torch.float16))):
        with pytest.raises(ValueError):
            sampler.logprobs_backward(x, r.rows, **bad)
    with pytest.raises(ValueError):
        sampler.logprobs_backward(x, r.rows[:3], grad_lse=g)


# ---- from hidden states ----

def lm_inputs(B, V, E, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn(B, E, generator=g, device="cuda") * 3
    norm = torch.rand(E, generator=g, device="cuda") + 0.5
    w = (torch.randn(V, E, generator=g, device="cuda") * (2.5 / math.sqrt(E))).to(torch.bfloat16)
    return hidden, norm, w


def lm_exact(hidden, norm, w, eps=1e-6):
    h = hidden.double()
    xn = (h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * norm.double()).float()
    xn = xn.to(torch.bfloat16).double()
    return xn @ w.double().t(), float((xn.abs() @ w.double().abs().t()).max())


@pytest.mark.parametrize("B,V,E,m", [(1, 1000, 64, 1), (3, 129, 72, 2), (16, 5003, 896, 1),
                                     (8, 1, 64, 1), (127, 300, 80, 1),
                                     (130, 4099, 256, 3), (513, 3001, 128, 1), (700, 20000, 64, 1),
                                     (4500, 700, 64, 1), (9000, 300, 64, 2), (6, 90, 12288, 1)])
def test_lmhead_logprobs(sampler, B, V, E, m):
    """The logits are f32 accumulations of exact products, 16 at a time: each of the E / 16
    steps (and one within) is off by at most a step, 2^-23, of the sum of magnitudes."""
    hidden, norm, w = lm_inputs(B, V, E)
    ids = some_ids(B, V, m)
    x, size = lm_exact(hidden, norm, w)
    for temp in (1.0, torch.linspace(0.5, 2.0, B, device="cuda")):
        r = sampler.lmhead_logprobs(hidden, norm, w, ids, temp=temp)
        sampler.check_device_status()
        it = torch.tensor([inv_temp(t) for t in (temp.tolist() if isinstance(temp, torch.Tensor)
                                                 else [temp] * B)], dtype=torch.float64, device="cuda")
        lse, h, logp, t_sum, t_lse, t_h = exact(x, it)
        off = (E / 16 + 2) * 2 ** -23 * size * it  # of a logit over temp
        e1 = (logp.exp() * (logp - logp.max(1, keepdim=True).values).abs()).sum(1)
        close(r.lse, lse, t_lse + off, "lse")
        close(r.entropy, h, t_h + 2 * off * (1 + e1), "entropy")
        inside = (ids >= 0) & (ids < V)
        want = torch.where(inside, torch.gather(logp, 1, ids.clamp(0, V - 1).long()), 0.0)
        close(r.logp, want, (t_sum + 2 * off)[:, None] + want.abs() * U, "logp")


def test_lmhead_logprobs_agrees_with_its_parts(sampler):
    """At 40 rows lmhead_logits takes the tensor cores too: the same logits."""
    hidden, norm, w = lm_inputs(40, 6001, 896, seed=3)
    ids = some_ids(40, 6001, 1)
    logits = sampler.lmhead_logits(hidden, norm, w)
    a = sampler.logprobs(logits, ids, temp=0.7)
    b = sampler.lmhead_logprobs(hidden, norm, w, ids, temp=0.7)
    size = lm_exact(hidden, norm, w)[1]
    tol = 2 * (896 / 16 + 2) * 2 ** -23 * size * inv_temp(0.7) + 4 * depth(6001) * U
    for name in ("logp", "lse", "entropy"):
        assert float((getattr(a, name) - getattr(b, name)).abs().max()) <= tol


def test_lmhead_logprobs_of_large_logits(sampler):
    """Logits of hundreds: the base of the sums has to move, by more than the exponential's
    range within a tile.  Tolerances as above (they grow with the logits)."""
    B, V, E = 40, 3000, 128
    hidden, norm, w = lm_inputs(B, V, E, seed=6)
    w = (w.float() * 60).to(torch.bfloat16)
    w[V - 1] *= 8
    ids = some_ids(B, V, 1)
    x, size = lm_exact(hidden, norm, w)
    lse, h, logp, t_sum, t_lse, t_h = exact(x, torch.ones(B, dtype=torch.float64, device="cuda"))
    r = sampler.lmhead_logprobs(hidden, norm, w, ids)
    off = (E / 16 + 2) * 2 ** -23 * size
    e1 = (logp.exp() * (logp - logp.max(1, keepdim=True).values).abs()).sum(1)
    close(r.lse, lse, t_lse + off, "lse")
    close(r.entropy, h, t_h + 2 * off * (1 + e1), "entropy")
    want = torch.where(ids >= 0, torch.gather(logp, 1, ids.clamp(min=0).long()), 0.0)
    close(r.logp, want, (t_sum + 2 * off)[:, None] + want.abs() * U, "logp")


@pytest.mark.parametrize("mode,B", [("single", 300), ("pair", 300), ("single", 2300), ("pair", 2300)])
def test_lmhead_logprobs_tiles(sampler, mode, B):
    hidden, norm, w = lm_inputs(B, 2500, 192, seed=4)
    ids = some_ids(B, 2500, 1)
    ref = sampler.lmhead_logprobs(hidden, norm, w, ids)
    sampler.set_lmhead_tiles(mode)
    try:
        r = sampler.lmhead_logprobs(hidden, norm, w, ids)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r2 = sampler.lmhead_logprobs(hidden, norm, w, ids)
        graph.replay()
        torch.cuda.synchronize()
    finally:
        sampler.set_lmhead_tiles("auto")
    for q in (r, r2):
        # the same logits; slices (and so the order of the sums) may differ
        for name in ("logp", "lse", "entropy"):
            assert float((getattr(q, name) - getattr(ref, name)).abs().max()) <= 4 * depth(2500) * U
    assert torch.equal(r.lse, r2.lse) and torch.equal(r.logp, r2.logp)


def test_lmhead_logprobs_refuses(sampler):
    hidden, norm, w = lm_inputs(4, 100, 64)
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    for a in ((hidden.double(), norm, w, ids), (hidden, norm[:32], w, ids), (hidden, norm, w.float(), ids),
              (hidden, norm, w, ids.long()), (hidden, norm, w[:, :32], ids), (hidden, norm, w.t(), ids)):
        with pytest.raises(ValueError):
            sampler.lmhead_logprobs(*a)
    assert sampler.lmhead_logprobs(hidden[:0], norm, w, ids[:0]).lse.shape == (0,)
