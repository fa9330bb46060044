"""The vocabulary-side operators beside the sampler: what is measured of each, in its
plain torch form and through the framework.

    logprobs         log probabilities of given tokens, entropy, log-sum-exp and the
                     top alternatives of every row of logits
    backward         their gradient with respect to the logits
    lmhead_logprobs  the same log probabilities from hidden states (rmsnorm, lm_head),
                     without the logits in memory
    embed            rows of the embedding table, scaled
    embed_backward   the gradient of the table, summed per token id

`own` is False for the plain forms and True for the framework's kernels.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6

_samplers = {}


def _sampler():
    """One handle per device, as a serving program keeps it."""
    from zeninfer_b200 import Sampler
    d = torch.cuda.current_device()
    if d not in _samplers:
        _samplers[d] = Sampler(d)
    return _samplers[d]


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one sequence being decoded: the id just drawn and five alternatives (latency)
        dict(name="logprobs_decode_1", op="logprobs", rows=1, vocab=151936, dtype="f32", ids=1,
             top=5, temp=0.7, mask=0.0),
        # a decode step of 256 sequences that asked for 20 alternatives each
        dict(name="logprobs_decode_256", op="logprobs", rows=256, vocab=151936, dtype="f32", ids=1,
             top=20, temp=0.7, mask=0.0),
        # constrained decoding: most columns masked, one row with nothing left, four
        # given tokens (answers to a choice), an odd vocabulary, so unaligned rows
        dict(name="logprobs_masked_61", op="logprobs", rows=61, vocab=50001, dtype="f16", ids=4,
             top=3, temp=1.0, mask=0.6),
        # scoring a prompt, or the forward half of a policy-gradient step
        dict(name="logprobs_score_4096", op="logprobs", rows=4096, vocab=151936, dtype="bf16",
             ids=1, top=0, temp=1.0, mask=0.0),
        # a small training step on masked f32 logits with unaligned rows
        dict(name="backward_ragged_333", op="backward", rows=333, vocab=50001, dtype="f32", ids=1,
             temp=0.8, mask=0.25),
        # a training step of 4096 tokens
        dict(name="backward_4096", op="backward", rows=4096, vocab=151936, dtype="bf16", ids=1,
             temp=1.0, mask=0.0),
        # the given ids of 16 running sequences, from their hidden states
        dict(name="lmhead_logprobs_16", op="lmhead_logprobs", rows=16, vocab=151936, embd=896,
             temp=1.0),
        # scoring 4096 prompt tokens from their hidden states
        dict(name="lmhead_logprobs_4096", op="lmhead_logprobs", rows=4096, vocab=151936, embd=896,
             temp=1.0),
        # the ids of a decode step, as f32 hidden states (latency)
        dict(name="embed_decode_64", op="embed", tokens=64, vocab=151936, embd=896, table="bf16",
             act="f32"),
        # a prompt batch
        dict(name="embed_prompt_32768", op="embed", tokens=32768, vocab=151936, embd=896,
             table="bf16", act="bf16"),
        # a small table trained in f32
        dict(name="embed_backward_1001", op="embed_backward", tokens=1001, vocab=32000, embd=640,
             table="f32", act="f32"),
        # a training step of 32,768 tokens with f32 gradients of a large table
        dict(name="embed_backward_32768", op="embed_backward", tokens=32768, vocab=151936,
             embd=896, table="f32", act="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "backward", "lmhead_logprobs", "embed", "embed_backward"])
    if op in ("logprobs", "backward"):
        c = dict(op=op, rows=_log_int(rng, 1, 2048), vocab=_log_int(rng, 1000, 151936),
                 dtype=rng.choice(["f32", "f16", "bf16"]), ids=rng.choice([1, 1, 2, 5]))
        if op == "logprobs":
            c["top"] = rng.choice([0, 1, 5, 20, 64])
        c["temp"] = rng.choice([1.0, 0.7, 1.3])
        c["mask"] = rng.choice([0.0, 0.0, 0.5, 0.95])
        return c
    if op == "lmhead_logprobs":
        return dict(op=op, rows=_log_int(rng, 1, 2048), vocab=_log_int(rng, 1000, 151936),
                    embd=8 * _log_int(rng, 8, 192), temp=rng.choice([1.0, 0.7, 1.3]))
    return dict(op=op, tokens=_log_int(rng, 1, 32768), vocab=_log_int(rng, 1000, 151936),
                embd=_log_int(rng, 64, 896), table=rng.choice(["f32", "f16", "bf16"]),
                act=rng.choice(["f32", "f16", "bf16"]))


# ---------------------------------------------------------------- inputs

def _token_ids(g, shape, vocab):
    """Ids with a natural-language-like frequency law, some of them -1 (a stopped row)."""
    u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    gone = torch.rand(shape, generator=g, device="cuda") < 0.02
    return torch.where(gone, -1, ids).to(torch.int32)


def _row_state(x, inv_temp):
    """[rows, 4] float32 (max, sum of exp((x - max) * inv_temp), entropy, inv_temp): what
    the forward pass keeps for the backward one.  In 64 bits, some rows at a time."""
    rows = torch.empty(x.shape[0], 4, dtype=torch.float32, device="cuda")
    for r in range(0, x.shape[0], 256):
        m, s, h, _ = _stats64(x[r:r + 256], inv_temp)
        rows[r:r + 256, 0], rows[r:r + 256, 1], rows[r:r + 256, 2] = m, s, h
    rows[:, 3] = inv_temp
    return rows


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    st = {"case": case}
    if op in ("logprobs", "backward"):
        B, V = case["rows"], case["vocab"]
        x = torch.randn(B, V, generator=g, device="cuda") * 2.5
        ids = _token_ids(g, (B, case["ids"]), V)
        # the given tokens are likely ones, as drawn or observed tokens are
        lift = torch.rand(B, case["ids"], generator=g, device="cuda") * 12.0
        x.scatter_add_(1, ids.clamp(min=0).long(), torch.where(ids >= 0, lift, 0.0))
        if case["mask"] > 0:
            x.masked_fill_(torch.rand(B, V, generator=g, device="cuda") < case["mask"], -math.inf)
            if B > 2:
                x[B // 2] = -math.inf
        st["logits"] = x.to(DTYPES[case["dtype"]])
        del x
        st["ids"] = ids
        if op == "backward":
            st["rows"] = _row_state(st["logits"], _inv_temp(case))
            st["g_logp"] = torch.randn(B, case["ids"], generator=g, device="cuda")
            st["g_entropy"] = torch.randn(B, generator=g, device="cuda") * 0.1
            st["g_lse"] = torch.randn(B, generator=g, device="cuda") * 0.1
    elif op == "lmhead_logprobs":
        B, V, E = case["rows"], case["vocab"], case["embd"]
        st["hidden"] = torch.randn(B, E, generator=g, device="cuda") * 3.0
        st["norm_w"] = torch.rand(E, generator=g, device="cuda") + 0.5
        st["weight"] = (torch.randn(V, E, generator=g, device="cuda")
                        * (2.5 / math.sqrt(E))).to(torch.bfloat16)
        st["ids"] = _token_ids(g, (B, 1), V)
    else:
        n, V, E = case["tokens"], case["vocab"], case["embd"]
        st["ids"] = _token_ids(g, (n,), V)
        if op == "embed":
            st["table"] = torch.randn(V, E, generator=g, device="cuda").to(DTYPES[case["table"]])
        else:
            st["grad"] = torch.randn(n, E, generator=g, device="cuda").to(DTYPES[case["act"]])
        st["scale"] = math.sqrt(E)
    return st


# ---------------------------------------------------------------- plain forms

def _inv_temp(case):
    """1 / temp in float32, as the sampler takes it."""
    return float(torch.ones((), dtype=torch.float32) / torch.tensor(case["temp"], dtype=torch.float32))


def _stats(x, inv_temp):
    """(max, sum, entropy, t = (x - max) * inv_temp, e = exp(t)) of float rows."""
    m = x.amax(1)
    t = (x - torch.where(torch.isinf(m), 0.0, m)[:, None]) * inv_temp
    e = torch.exp(t)
    s = e.sum(1)
    w = torch.where(e > 0, e * t, 0.0).sum(1)
    some = s > 0
    safe = torch.where(some, s, 1.0)
    h = torch.where(some, torch.log(safe) - w / safe, 0.0)
    return m, s, h, t, e


def _given(t, s, ids):
    """log p of the given ids ([rows, m]); 0 where the id is none."""
    got = torch.gather(t, 1, ids.clamp(min=0).long()) - torch.log(s)[:, None]
    got = torch.where((s > 0)[:, None], got, -math.inf)
    return torch.where(ids >= 0, got, 0.0)


def _order_keys(x):
    """int64 keys in the order of the values, the lower index first among equals."""
    u = (x + 0.0).view(torch.int32).long()
    u = torch.where(u < 0, -(u & 0x7FFFFFFF), u)
    return u * (1 << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))


def _plain_logprobs(x, ids, inv_temp, top):
    x = x.float()
    m, s, h, t, _ = _stats(x, inv_temp)
    out = {"logp": _given(t, s, ids), "entropy": h, "lse": m * inv_temp + torch.log(s)}
    if top:
        keys = torch.topk(_order_keys(x), top, dim=1).values
        at = x.shape[1] - 1 - (keys & 0xFFFFFFFF)
        out["top_ids"] = at.to(torch.int32)
        out["top_logp"] = _given(t, s, out["top_ids"])
    return out


def _plain_backward(st):
    x, ids, rows = st["logits"].float(), st["ids"].long(), st["rows"]
    m, s, h, inv_temp = rows[:, 0], rows[:, 1], rows[:, 2], rows[:, 3]
    some = s > 0
    t = (x - torch.where(some, m, 0.0)[:, None]) * inv_temp[:, None]
    safe = torch.where(some, s, 1.0)
    p = torch.exp(t) / safe[:, None] * some[:, None]
    logp = t - torch.log(safe)[:, None]
    given = (ids >= 0) & some[:, None]
    gl = torch.where(given, st["g_logp"], 0.0)
    d = p * (st["g_lse"] - gl.sum(1) - st["g_entropy"] * h)[:, None]
    d = d - torch.where(p > 0, p * logp, 0.0) * st["g_entropy"][:, None]
    d.scatter_add_(1, ids.clamp(min=0), gl)
    return (d * inv_temp[:, None]).to(st["logits"].dtype)


def _normed(hidden, norm_w, dtype):
    """rmsnorm in 64 bits, rounded to float32 and then bfloat16 (values next to a border)."""
    x = hidden.double()
    xn = x / torch.sqrt(x.square().mean(1, keepdim=True) + EPS) * norm_w.double()
    return xn.float().to(torch.bfloat16).to(dtype)


def _plain(st):
    case = st["case"]
    op = case["op"]
    if op == "logprobs":
        return _plain_logprobs(st["logits"], st["ids"], _inv_temp(case), case["top"])
    if op == "backward":
        return _plain_backward(st)
    if op == "lmhead_logprobs":
        xn = _normed(st["hidden"], st["norm_w"], torch.float32)
        logits = xn @ st["weight"].float().t()
        return _plain_logprobs(logits, st["ids"], _inv_temp(case), 0)
    ids = st["ids"].long()
    if op == "embed":
        rows = st["table"][ids.clamp(min=0)].float() * st["scale"]
        return torch.where((ids >= 0)[:, None], rows, 0.0).to(DTYPES[case["act"]])
    grad = torch.where((ids >= 0)[:, None], st["grad"].float(), 0.0)
    table = torch.zeros(case["vocab"], case["embd"], device=grad.device)
    table.index_add_(0, ids.clamp(min=0), grad)
    return (table * st["scale"]).to(DTYPES[case["table"]])


def run(st):
    if not own:
        return _plain(st)
    case, s = st["case"], _sampler()
    op = case["op"]
    if op == "logprobs":
        r = s.logprobs(st["logits"], st["ids"], temp=case["temp"], top=case["top"])
        out = {"logp": r.logp, "entropy": r.entropy, "lse": r.lse}
        if case["top"]:
            out["top_ids"], out["top_logp"] = r.top_ids, r.top_logp
        return out
    if op == "backward":
        return s.logprobs_backward(st["logits"], st["rows"], st["ids"], grad_logp=st["g_logp"],
                                   grad_entropy=st["g_entropy"], grad_lse=st["g_lse"])
    if op == "lmhead_logprobs":
        r = s.lmhead_logprobs(st["hidden"], st["norm_w"], st["weight"], st["ids"],
                              temp=case["temp"], eps=EPS)
        return {"logp": r.logp, "entropy": r.entropy, "lse": r.lse}
    if op == "embed":
        return s.embed(st["table"], st["ids"], scale=st["scale"], out_dtype=DTYPES[case["act"]])
    return s.embed_backward(st["grad"], st["ids"], case["vocab"], scale=st["scale"],
                            dtype=DTYPES[case["table"]])


# ---------------------------------------------------------------- what a pass has to do

def work(case):
    op = case["op"]
    if op in ("logprobs", "backward"):
        B, V, m = case["rows"], case["vocab"], case["ids"]
        one = B * V * SIZES[case["dtype"]]
        if op == "logprobs":
            return {"bytes": one + B * (8 * m + 8 * case["top"] + 8), "flops": 4 * B * V}
        return {"bytes": 2 * one + B * (8 * m + 24), "flops": 6 * B * V}
    if op == "lmhead_logprobs":
        B, V, E = case["rows"], case["vocab"], case["embd"]
        return {"bytes": 2 * V * E + 4 * B * E + 4 * E + 16 * B, "flops": 2 * B * V * E}
    n, V, E = case["tokens"], case["vocab"], case["embd"]
    t, a = SIZES[case["table"]], SIZES[case["act"]]
    if op == "embed":
        return {"bytes": min(n, V) * E * t + n * E * a + 4 * n, "flops": n * E}
    return {"bytes": V * E * t + n * E * a + 4 * n, "flops": n * E}


# ---------------------------------------------------------------- 64-bit values

def _stats64(x, inv_temp):
    """(max, sum, entropy, log-sum-exp) of rows in 64 bits, by torch's logsumexp."""
    z = x.double() * inv_temp
    lse = torch.logsumexp(z, 1)
    m = x.double().max(1).values
    dead = torch.isneginf(lse)
    logp = z - torch.where(dead, 0.0, lse)[:, None]
    p = torch.exp(logp)
    h = -(p * torch.nan_to_num(logp, neginf=0.0)).sum(1)
    s = torch.where(dead, 0.0, torch.exp(lse - torch.where(dead, 0.0, m) * inv_temp))
    return m, s, h, lse


def _pick64(x, inv_temp, lse, ids):
    z = torch.gather(x.double() * inv_temp, 1, ids.clamp(min=0).long())
    got = torch.where(torch.isneginf(lse)[:, None], -math.inf, z - lse[:, None])
    return got.masked_fill(ids < 0, 0.0)


def _exact_rows(x, ids, inv_temp, top):
    _, _, h, lse = _stats64(x, inv_temp)
    out = {"logp": _pick64(x, inv_temp, lse, ids), "entropy": h, "lse": lse}
    if top:
        v = torch.sort(x.double(), dim=1, descending=True).values[:, :top] * inv_temp
        out["top_ids"] = None
        out["top_logp"] = torch.where(torch.isneginf(lse)[:, None], -math.inf, v - lse[:, None])
    return out


def _stack(parts):
    return {k: None if parts[0][k] is None else torch.cat([p[k] for p in parts]) for k in parts[0]}


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "logprobs":
        return _stack([_exact_rows(st["logits"][r:r + 128], st["ids"][r:r + 128], _inv_temp(case),
                                   case["top"]) for r in range(0, case["rows"], 128)])
    if op == "lmhead_logprobs":
        xn = _normed(st["hidden"], st["norm_w"], torch.float64)
        w = st["weight"].double()
        return _stack([_exact_rows(xn[r:r + 128] @ w.t(), st["ids"][r:r + 128], _inv_temp(case), 0)
                       for r in range(0, case["rows"], 128)])
    if op == "backward":
        out = torch.empty(st["logits"].shape, dtype=torch.float64, device="cuda")
        it = _inv_temp(case)
        for r in range(0, case["rows"], 128):
            x, ids = st["logits"][r:r + 128], st["ids"][r:r + 128]
            _, _, h, lse = _stats64(x, it)
            dead = torch.isneginf(lse)
            logp = x.double() * it - torch.where(dead, 0.0, lse)[:, None]
            p = torch.exp(logp)
            gh, gz = (st[k][r:r + 128].double()[:, None] for k in ("g_entropy", "g_lse"))
            d = gz * p - gh * p * (torch.nan_to_num(logp, neginf=0.0) + h[:, None])
            gl = st["g_logp"][r:r + 128].double() * (ids >= 0) * ~dead[:, None]
            for j in range(ids.shape[1]):
                at = torch.zeros_like(p).scatter_(1, ids[:, j:j + 1].clamp(min=0).long(), 1.0)
                d += gl[:, j:j + 1] * (at - p)
            out[r:r + 128] = d * it
        return out
    ids = st["ids"].long()
    live = (ids >= 0).double()[:, None]
    if op == "embed":
        return torch.nn.functional.embedding(ids.clamp(min=0), st["table"]).double() * live * st["scale"]
    out = torch.zeros(case["vocab"] + 1, case["embd"], dtype=torch.float64, device="cuda")
    order = torch.argsort(ids, stable=True)
    out.index_put_((torch.where(ids < 0, case["vocab"], ids)[order],), st["grad"].double()[order],
                   accumulate=True)
    return out[:case["vocab"]] * st["scale"]
