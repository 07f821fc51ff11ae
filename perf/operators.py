"""What is measured of the operators between the QKV projection and the optimizer step: attention on the fused QKV tensor
(forward, and the backward pass that recomputes the probabilities) and the log probabilities of given tokens with entropy
and top alternatives (forward and gradient).  Shapes are those of this repository's tests and benchmark (head layouts of the
0.5B, 1.5B and 7B configurations at 8192 tokens) or generic ones.

`run` computes the operators from elementary torch operations in 32 bits where `own` is false, and calls the framework's
kernels where it is true; `exact` computes them from their definitions in 64 bits."""
import math
import random

import torch

own = False

TOPK_MAX = 32
HEADS = [(14, 2), (12, 2), (28, 4), (8, 8), (6, 1), (9, 3)]          # (query heads, key/value heads)
HEAD_DIMS = [32, 64, 80, 96, 128]


def listed():
    def att(name, op, B, T, Nq, Nkv, HD, mask, span=0):
        return {"name": name, "op": op, "B": B, "T": T, "Nq": Nq, "Nkv": Nkv, "HD": HD, "mask": mask, "span": span}

    def lp(name, op, N, V, P, dtype, topk, entropy, banned=False):
        return {"name": name, "op": op, "N": N, "V": V, "P": P, "dtype": dtype, "topk": topk, "entropy": entropy, "banned": banned}

    return [
        # one short prompt through the 0.5B model's heads: a call whose launch counts
        att("attention fwd 1x40", "attention_forward", 1, 40, 14, 2, 64, "causal"),
        # the benchmark's 8192 tokens as eight sequences of 1024 through the 7B model's heads
        att("attention fwd 8x1024", "attention_forward", 8, 1024, 28, 4, 128, "causal"),
        # documents packed into rows of odd length, 1.5B heads
        att("attention fwd docs 3x2711", "attention_forward", 3, 2711, 12, 2, 128, "documents", 700),
        # the same 8192 tokens as one long sequence
        att("attention fwd 1x8192", "attention_forward", 1, 8192, 28, 4, 128, "causal"),
        # backward of a short odd batch padded on the left (rows that may look at nothing)
        att("attention bwd pad 2x129", "attention_backward", 2, 129, 14, 2, 64, "padded", 45),
        # backward of the benchmark's batch
        att("attention bwd 8x1024", "attention_backward", 8, 1024, 28, 4, 128, "causal"),
        # backward of long rows with a sliding window, 0.5B heads
        att("attention bwd window 1x8192", "attention_backward", 1, 8192, 14, 2, 64, "window", 1500),
        # one sequence served: the next token's alternatives, some tokens banned
        lp("logprobs 1x151936 top20", "token_logprobs", 1, 151936, 151936, "bf16", 20, False, True),
        # scoring a batch of sampled tokens with entropy and top alternatives
        lp("logprobs 4096x151936 top5", "token_logprobs", 4096, 151936, 151936, "bf16", 5, True),
        # fp32 logits with an odd vocabulary and odd rows
        lp("logprobs 777x50257 f32", "token_logprobs", 777, 50257, 50257, "f32", 0, True),
        # gradient of the training loss over one chunk of the batch
        lp("logprobs bwd 4096x151936", "token_logprobs_backward", 4096, 151936, 151936, "bf16", 0, False),
        # policy gradient with an entropy term on fp32 logits, vocabulary padded
        lp("logprobs bwd 777x50257 f32", "token_logprobs_backward", 777, 50257, 50304, "f32", 0, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    if rng.random() < 0.55:
        while True:
            (Nq, Nkv), HD = rng.choice(HEADS), rng.choice(HEAD_DIMS)
            B, T = _log_int(rng, 1, 8), _log_int(rng, 1, 8192)
            if B * Nq * T * T <= 28 * 8192 * 8192 and B * T <= 16384:
                break
        mask = rng.choice(["causal", "documents", "window", "padded"])
        span = 0 if mask == "causal" else _log_int(rng, 1, max(1, T if mask != "padded" else (T + 1) // 2))
        return {"op": rng.choice(["attention_forward", "attention_backward"]), "B": B, "T": T, "Nq": Nq, "Nkv": Nkv, "HD": HD,
                "mask": mask, "span": span}
    dtype = rng.choice(["bf16", "f32"])
    while True:
        N, V = _log_int(rng, 1, 8192), _log_int(rng, 64, 262144)
        if N * V <= 4096 * 151936 // (2 if dtype == "f32" else 1):
            break
    op = rng.choice(["token_logprobs", "token_logprobs_backward"])
    P = V + rng.choice([0, 0, 0, 1, 7, 64])
    topk = rng.choice([0, 1, 5, 20, TOPK_MAX]) if op == "token_logprobs" else 0
    return {"op": op, "N": N, "V": V, "P": P, "dtype": dtype, "topk": topk, "entropy": rng.random() < 0.5, "banned": rng.random() < 0.3}


# ---- masks ------------------------------------------------------------------------------------------------------------
def _first_keys(case):
    """[B][T] list of the first key each query may look at, or None for the plain causal mask: a function of the case alone,
    so that `work` can count the pairs."""
    B, T, mask, span = case["B"], case["T"], case["mask"], case["span"]
    if mask == "causal":
        return None
    rows = []
    for b in range(B):
        r = random.Random(1000 * T + 10 * span + b)
        if mask == "window":
            row = [max(0, t - span + 1) for t in range(T)]
        elif mask == "padded":                                  # the first tokens are padding and may look at nothing
            pad = min(T, r.randint(0, span))
            row = [T] * pad + [pad] * (T - pad)
        else:                                                   # documents of `span` tokens on average
            row = []
            while len(row) < T:
                row += [len(row)] * max(1, min(int(r.expovariate(1.0 / span)) + 1, T - len(row)))
        rows.append(row)
    return rows


def _pairs(case):
    T, rows = case["T"], _first_keys(case)
    if rows is None:
        return case["B"] * T * (T + 1) // 2
    return sum(max(0, t + 1 - f) for row in rows for t, f in enumerate(row))


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, g, std=1.0):
    return torch.randn(shape, device="cuda", generator=g) * std


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["op"].startswith("attention"):
        B, T, Nq, Nkv, HD = (case[n] for n in ("B", "T", "Nq", "Nkv", "HD"))
        # projections of normalised activations: unit-scale queries and keys, a few strong directions in them
        x = _normal((B, T, (Nq + 2 * Nkv) * HD), g)
        x[..., ::29] *= 2.0
        s["qkv"] = x.to(torch.bfloat16)
        rows = _first_keys(case)
        s["first_key"] = None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda")
        if case["op"] == "attention_forward":
            s["out"] = torch.empty((B, T, Nq * HD), dtype=torch.bfloat16, device="cuda")
            s["lse"] = torch.empty((B, Nq, T), device="cuda")
        else:
            s["dout"] = _normal((B, T, Nq * HD), g, 1e-2).to(torch.bfloat16)
            s["out"], s["lse"] = _attention(s)               # what the forward pass left
            s["dqkv"] = torch.empty_like(s["qkv"])
        return s
    N, V, P = case["N"], case["V"], case["P"]
    x = _normal((N, P), g, 2.5)
    s["targets"] = torch.randint(0, V, (N,), device="cuda", generator=g, dtype=torch.int32)
    # the model likes most of the given tokens; one target in sixteen is ignored (prompt or padding)
    x.scatter_add_(1, s["targets"].long()[:, None], 6.0 + _normal((N, 1), g, 3.0))
    if case["banned"]:
        x.masked_fill_(torch.rand((N, P), device="cuda", generator=g) < 0.3, float("-inf"))
        x.scatter_(1, s["targets"].long()[:, None], 4.0)
    if N > 1:
        s["targets"][torch.rand(N, device="cuda", generator=g) < 1 / 16] = -100
    s["logits"] = x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    f32 = lambda *shape: torch.empty(shape, device="cuda")  # noqa: E731
    if case["op"] == "token_logprobs":
        s["logp"], s["lse"] = f32(N), f32(N)
        s["entropy_out"] = f32(N) if case["entropy"] else None
        s["top_logp"] = f32(N, case["topk"]) if case["topk"] else None
        s["top_ids"] = torch.empty((N, case["topk"]), dtype=torch.int32, device="cuda") if case["topk"] else None
    else:
        del x
        s["lse"], s["entropy_in"] = _statistics(s["logits"][:, :V].float())
        s["dlogp"] = _normal((N,), g) / N
        s["dentropy"] = torch.full((N,), 1e-2 / N, device="cuda") if case["entropy"] else None
        s["dlogits"] = torch.empty_like(s["logits"])
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _heads(s, dtype=torch.float32):
    """q [B, Nkv, G*T, HD] (the G query heads of each key/value head one after the other), k and v [B, Nkv, T, HD]."""
    B, T, Nq, Nkv, HD = (s[n] for n in ("B", "T", "Nq", "Nkv", "HD"))
    x = s["qkv"].to(dtype).view(B, T, Nq + 2 * Nkv, HD).transpose(1, 2)
    q, k, v = x[:, :Nq], x[:, Nq:Nq + Nkv], x[:, Nq + Nkv:]
    return q.reshape(B, Nkv, (Nq // Nkv) * T, HD).contiguous(), k.contiguous(), v.contiguous()


def _allowed(s):
    """Truth values [B or 1, 1, 1, T, T]: may query t look at key k."""
    T = s["T"]
    at = torch.arange(T, device="cuda")
    allowed = (at[None, :] <= at[:, None])[None]
    if s["first_key"] is not None:
        allowed = allowed & (at[None, None, :] >= s["first_key"][:, :, None])
    return allowed[:, None, None]


def _scores(s, q, k):
    B, T, Nq, Nkv = (s[n] for n in ("B", "T", "Nq", "Nkv"))
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, Nkv, Nq // Nkv, T, T)
    return x.mul_(1.0 / math.sqrt(s["HD"])).masked_fill_(~_allowed(s), float("-inf"))


def _merge(x, s):
    """[B, Nkv, G*T, HD] -> [B, T, Nq, HD]"""
    return x.reshape(s["B"], s["Nq"], s["T"], s["HD"]).transpose(1, 2)


def _attention(s):
    B, T, Nq, Nkv, HD = (s[n] for n in ("B", "T", "Nq", "Nkv", "HD"))
    q, k, v = _heads(s)
    x = _scores(s, q, k)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    x = x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True)
    lse = m + total.log()
    x = x.div_(torch.where(total == 0, 1.0, total))
    out = _merge(torch.matmul(x.view(B, Nkv, (Nq // Nkv) * T, T), v), s)
    return out.reshape(B, T, Nq * HD).to(torch.bfloat16), lse.reshape(B, Nq, T).contiguous()


def _attention_gradient(s):
    B, T, Nq, Nkv, HD = (s[n] for n in ("B", "T", "Nq", "Nkv", "HD"))
    G = Nq // Nkv
    q, k, v = _heads(s)
    lse = s["lse"].view(B, Nkv, G, T, 1)
    p = _scores(s, q, k)
    p = p.sub_(torch.where(lse == float("-inf"), 0.0, lse)).exp_().view(B, Nkv, G * T, T)
    dout = s["dout"].float().view(B, T, Nq, HD).transpose(1, 2).reshape(B, Nkv, G * T, HD).contiguous()
    out = s["out"].float().view(B, T, Nq, HD).transpose(1, 2).reshape(B, Nkv, G * T, HD)
    delta = (dout * out).sum(-1, keepdim=True)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), dout)
    ds = torch.matmul(dout, v.transpose(2, 3).contiguous()).sub_(delta).mul_(p).mul_(1.0 / math.sqrt(HD))
    del p
    dq = _merge(torch.matmul(ds, k), s)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    grad = torch.cat([dq, dk.transpose(1, 2), dv.transpose(1, 2)], dim=2)
    return grad.reshape(B, T, (Nq + 2 * Nkv) * HD).to(torch.bfloat16)


def _statistics(x):
    """(lse, entropy) of rows of logits in x's type."""
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1)
    part = torch.where(e > 0, (x - m) * e, 0.0).sum(-1)
    return m[:, 0] + total.log(), total.log() - part / total


def _logprobs(s):
    x = s["logits"][:, :s["V"]].float()
    lse, entropy = _statistics(x)
    t = s["targets"].long()
    given = (t >= 0) & (t < s["V"])
    logp = torch.where(given, x.gather(1, torch.where(given, t, 0)[:, None])[:, 0] - lse, 0.0)
    got = {"logp": logp, "lse": lse}
    if s["entropy"]:
        got["entropy"] = entropy
    if s["topk"]:
        val, ids = torch.sort(x, dim=1, descending=True, stable=True)
        got["top_logp"] = val[:, :s["topk"]] - lse[:, None]
        got["top_ids"] = ids[:, :s["topk"]].to(torch.int32)
    return got


def _logprobs_gradient(s):
    V = s["V"]
    x = s["logits"][:, :V].float()
    t = s["targets"].long()
    given = (t >= 0) & (t < V)
    g = torch.where(given, s["dlogp"], 0.0)
    d = x - s["lse"][:, None]
    p = d.exp()
    grad = p * -g[:, None]
    if s["dentropy"] is not None:
        grad -= torch.where(p > 0, p * (d + s["entropy_in"][:, None]), 0.0) * s["dentropy"][:, None]
    grad.scatter_add_(1, torch.where(given, t, 0)[:, None], g[:, None])
    full = torch.zeros((s["N"], s["P"]), dtype=s["logits"].dtype, device="cuda")
    full[:, :V] = grad
    return full


# ---- one pass ---------------------------------------------------------------------------------------------------------
def _scratch(s, size):
    """The workspace a program allocates once and keeps."""
    if "scratch" not in s:
        s["scratch"] = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    return s["scratch"]


def run(s):
    op = s["op"]
    if not own:
        if op == "attention_forward":
            out, lse = _attention(s)
            return {"out": out, "lse": lse}
        if op == "attention_backward":
            return {"dqkv": _attention_gradient(s)}
        return _logprobs(s) if op == "token_logprobs" else {"dlogits": _logprobs_gradient(s)}
    from llmq_amd import kernels as K
    if op == "attention_forward":
        K.attention_forward(s["out"], s["lse"], s["qkv"], None, s["Nq"], s["Nkv"], s["first_key"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "attention_backward":
        size = K.get_attention_backward_scratch_size(s["B"], s["T"], s["Nq"], s["Nkv"], s["HD"])
        K.attention_backward(s["dqkv"], s["dout"], s["out"], s["lse"], s["qkv"], _scratch(s, size), s["Nq"], s["Nkv"],
                             s["first_key"])
        return {"dqkv": s["dqkv"]}
    if op == "token_logprobs":
        size = K.get_token_logprobs_scratch_size(s["N"], s["V"], s["topk"])
        K.token_logprobs(s["logp"], s["entropy_out"], s["lse"], s["top_logp"], s["top_ids"], s["logits"], s["targets"],
                         _scratch(s, size), s["V"])
        got = {"logp": s["logp"], "lse": s["lse"]}
        if s["entropy"]:
            got["entropy"] = s["entropy_out"]
        if s["topk"]:
            got["top_logp"], got["top_ids"] = s["top_logp"], s["top_ids"]
        return got
    K.token_logprobs_backward(s["dlogits"], s["dlogp"], s["dentropy"], s["logits"], s["targets"], s["lse"],
                              s["entropy_in"], None, s["V"])
    return {"dlogits": s["dlogits"]}


def work(case):
    if case["op"].startswith("attention"):
        B, T, Nq, Nkv, HD = (case[n] for n in ("B", "T", "Nq", "Nkv", "HD"))
        qkv, o, lse = 2 * B * T * (Nq + 2 * Nkv) * HD, 2 * B * T * Nq * HD, 4 * B * T * Nq
        mask = 0 if case["mask"] == "causal" else 4 * B * T
        pairs = _pairs(case) * Nq * HD
        if case["op"] == "attention_forward":
            return {"bytes": qkv + o + lse + mask, "flops": 4 * pairs}
        return {"bytes": 2 * qkv + 2 * o + lse + mask, "flops": 10 * pairs}
    N, V, P = case["N"], case["V"], case["P"]
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "token_logprobs":
        return {"bytes": N * V * es + N * (12 + 4 * case["entropy"] + 8 * case["topk"]), "flops": 6 * N * V}
    return {"bytes": N * (V + P) * es + N * (12 + 8 * case["entropy"]), "flops": 6 * N * V}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _exact_attention(s, gradient):
    """Head by head; the gradient from the definition (out and lse in 64 bits too)."""
    B, T, Nq, Nkv, HD = (s[n] for n in ("B", "T", "Nq", "Nkv", "HD"))
    x = s["qkv"].double().view(B, T, Nq + 2 * Nkv, HD)
    res = torch.zeros((B, T, Nq + 2 * Nkv if gradient else Nq, HD), dtype=torch.float64, device="cuda")
    lses = torch.zeros((B, Nq, T), dtype=torch.float64, device="cuda")
    do = s["dout"].double().view(B, T, Nq, HD) if gradient else None
    idx = torch.arange(T, device="cuda")
    for b in range(B):
        lo = torch.zeros(T, dtype=torch.int64, device="cuda") if s["first_key"] is None else s["first_key"][b].long()
        banned = (idx[None, :] > idx[:, None]) | (idx[None, :] < lo[:, None])
        for h in range(Nq):
            kv = h // (Nq // Nkv)
            q, k, v = x[b, :, h], x[b, :, Nq + kv], x[b, :, Nq + Nkv + kv]
            a = (q @ k.T) / math.sqrt(HD)
            a[banned] = float("-inf")
            lse = torch.logsumexp(a, dim=1)
            lses[b, h] = lse
            a = torch.exp(a - lse[:, None].clamp_min(-1e300))
            if not gradient:
                res[b, :, h] = a @ v
                continue
            da = do[b, :, h] @ v.T
            res[b, :, Nq + Nkv + kv] += a.T @ do[b, :, h]
            a *= (da - (a * da).sum(1, keepdim=True)) / math.sqrt(HD)
            res[b, :, h] = a @ k
            res[b, :, Nq + kv] += a.T @ q
    res = res.reshape(B, T, -1)
    return {"dqkv": res} if gradient else {"out": res, "lse": lses}


def _exact_rows(s, lo, hi):
    x = s["logits"][lo:hi, :s["V"]].double()
    logp = torch.log_softmax(x, dim=1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(1)
    t = s["targets"][lo:hi].long()
    given = (t >= 0) & (t < s["V"])
    safe = torch.where(given, t, 0)[:, None]
    if s["op"] == "token_logprobs":
        got = {"logp": torch.where(given, logp.gather(1, safe)[:, 0], 0.0), "lse": torch.logsumexp(x, dim=1)}
        if s["entropy"]:
            got["entropy"] = entropy
        if s["topk"]:
            got["top_logp"] = torch.sort(logp, dim=1, descending=True)[0][:, :s["topk"]]
        return got
    g = torch.where(given, s["dlogp"][lo:hi].double(), 0.0)
    grad = torch.zeros((hi - lo, s["P"]), dtype=torch.float64, device="cuda")
    grad[:, :s["V"]] = -g[:, None] * p
    if s["dentropy"] is not None:
        grad[:, :s["V"]] -= s["dentropy"][lo:hi].double()[:, None] * (plogp + p * entropy[:, None])
    grad.scatter_add_(1, safe, g[:, None])
    return {"dlogits": grad}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("attention"):
        return _exact_attention(s, case["op"] == "attention_backward")
    step = max(1, (1 << 28) // case["P"])
    parts = [_exact_rows(s, lo, min(case["N"], lo + step)) for lo in range(0, case["N"], step)]
    got = {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
    if case["topk"]:
        got["top_ids"] = None                                   # whole numbers: held to the plain form's
    return got
