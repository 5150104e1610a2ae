"""Measured cases of the batched serving operators: a paged key-value cache's
append, the attention that reads it, and the verification of drafted tokens.

* ``append``: q/k RMSNorm and rotary embedding of the merged q/k/v projection,
  keys and values written into their cache slots (`paged_append`).
* ``attention``: attention of the newest token, or of a few drafted ones, of each
  sequence over its pages (`paged_attention`).
* ``verify``: acceptance of drafted tokens against the target's distribution and
  the draw of the token after them (`speculative_verify`).

`run` with `own` false computes the operators in plain torch (32-bit arithmetic,
one rounding at the end); with `own` true it calls the framework's operators.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
THETA = 1e6
MAX_POS = 1 << 17
FLT_MAX = torch.finfo(torch.float32).max


# ------------------------------------------------------------------ the cases
def listed():
    """8B-shaped heads (32 query, 8 key-value, 128 wide) where nothing else is said."""
    return [
        # one sequence's next four drafted tokens: the smallest append, all latency
        _append("append-4-tokens", T=4),
        # a batch of 24 sequences verifying 8 tokens each, keys stored token-major
        _append("append-192-tokens", T=192, layout="nhd", skip=0.1),
        # a long prompt chunk, some of its rows padding
        _append("append-8192-tokens", T=8192, skip=0.02),
        # a small draft model's heads, 64 wide, half of them rotated, no q/k norm, pages of 24
        _append("append-odd-fp16", T=333, Hq=14, Hk=2, D=64, R=32, ps=24, norm=False, dtype="fp16"),
        # one short conversation, one new token: the smallest read, all latency
        _attention("attend-1x100", B=1, L=1, lo=100, hi=100),
        # an ordinary serving batch, ragged, one new token each
        _attention("attend-32x2k", B=32, L=1, lo=300, hi=4096),
        # two long documents: the cache's length has to be split over the whole GPU
        _attention("attend-2x128k", B=2, L=1, lo=120000, hi=131072, ps=64),
        # verification of 8 drafted rows per sequence under a block mask
        _attention("attend-verify-16x8", B=16, L=8, lo=1000, hi=3000, mask="tail"),
        # a draft model's heads: 7 query heads per key head, 64 wide, pages of 24, some rows empty
        _attention("attend-odd-fp16", B=19, L=1, lo=1, hi=1500, Hq=14, Hk=2, D=64, ps=24, dtype="fp16",
                   layout="nhd", empty=0.1),
        # one sequence, drafts without probabilities (greedy drafting), a small vocabulary
        _verify("verify-1x4", B=1, K=4, V=32000, draft="tokens"),
        # an ordinary batch, sampled drafts, temperatures of their own, an odd vocabulary, 32-bit logits
        _verify("verify-12x3-odd", B=12, K=3, V=50021, dtype="fp32", temp="mixed", ragged=True),
        # a large batch over the 8B model's vocabulary
        _verify("verify-64x7", B=64, K=7, V=151936),
    ]


def _append(name=None, **kw):
    return _case(name, dict(op="append", T=1, Hq=32, Hk=8, D=128, R=kw.get("D", 128), ps=16, norm=True, dtype="bf16",
                            layout="hnd", skip=0.0), kw)


def _attention(name=None, **kw):
    return _case(name, dict(op="attention", B=1, L=1, lo=1, hi=1, Hq=32, Hk=8, D=128, ps=16, dtype="bf16",
                            layout="hnd", mask="causal", empty=0.0), kw)


def _verify(name=None, **kw):
    return _case(name, dict(op="verify", B=1, K=1, V=1, dtype="bf16", draft="logits", temp="one", ragged=False), kw)


def _case(name, base, kw):
    base.update(kw)
    if name is not None:
        base["name"] = name
    return base


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "verify"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "verify":
        V = rng.choice([151936, 32000, _log_int(rng, 1000, 151936)])
        K = rng.randint(1, 8)
        B = _log_int(rng, 1, max(1, min(64, 64 * 8 * 151936 // (V * (K + 1)))))
        return _verify(B=B, K=K, V=V, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]) if B * K < 200 else dtype,
                       draft=rng.choice(["logits", "logits", "tokens"]), temp=rng.choice(["one", "mixed"]),
                       ragged=rng.random() < 0.5)
    D = rng.choice([128, 128, 64])
    Hk = rng.choice([1, 2, 4, 8, 8])
    Hq = Hk * rng.choice([1, 2, 4, 4, 5, 7, 8])
    ps = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    layout = rng.choice(["hnd", "nhd"])
    if op == "append":
        return _append(T=_log_int(rng, 1, 8192 if Hq + 2 * Hk <= 48 else 4096), Hq=Hq, Hk=Hk, D=D,
                       R=rng.choice([D, D, D // 2]), ps=ps, norm=rng.random() < 0.7, dtype=dtype, layout=layout,
                       skip=rng.choice([0.0, 0.1]))
    B = _log_int(rng, 1, 128)
    hi = _log_int(rng, 8, max(8, min(131072, (1 << 28) // (B * Hk * D))))
    return _attention(B=B, L=rng.choice([1, 1, 1, 2, 4, 5, 8, 16]), lo=_log_int(rng, 1, hi), hi=hi, Hq=Hq, Hk=Hk, D=D,
                      ps=ps, dtype=dtype, layout=layout, mask=rng.choice(["causal", "tail"]),
                      empty=rng.choice([0.0, 0.1]))


def _lengths(c):
    """The case's key counts: the same multiset for every seed, so that its work is the case's own."""
    r = random.Random(c["B"] * 7919 + c["hi"])
    n = [_log_int(r, c["lo"], c["hi"]) for _ in range(c["B"])]
    n[0] = c["hi"]
    return [0 if i > 0 and r.random() < c["empty"] else v for i, v in enumerate(n)]


def _draft_counts(c):
    r = random.Random(c["B"] * 31 + c["K"])
    return [r.randint(0, c["K"]) if c["ragged"] else c["K"] for _ in range(c["B"])]


def work(c):
    e = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "append":
        T, D, H = c["T"], c["D"], c["Hq"] + 2 * c["Hk"]
        # the projections read, q and the new keys and values written, one table row and two indices a token
        return {"bytes": T * (2 * H * D * e + c["R"] * 4 + 16), "flops": T * (c["Hq"] + c["Hk"]) * (3 * c["R"] + 4 * D)}
    if c["op"] == "attention":
        n = _lengths(c)
        kv = sum(n) * c["Hk"] * c["D"] * 2 * e
        qo = c["B"] * c["L"] * c["Hq"] * (2 * c["D"] * e + 4)
        pages = sum(-(-v // c["ps"]) for v in n) * 4
        return {"bytes": kv + qo + pages, "flops": 4 * sum(n) * c["L"] * c["Hq"] * c["D"]}
    d = _draft_counts(c)
    rows = sum(d) + c["B"] + (sum(d) if c["draft"] == "logits" else 0)
    return {"bytes": rows * c["V"] * e + c["B"] * c["V"] * 4, "flops": 4 * rows * c["V"]}


# ------------------------------------------------------------------ inputs
def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    r = random.Random(int(seed))
    s = dict(c)
    s.pop("name", None)
    if c["op"] == "append":
        _prepare_append(c, s, g)
    elif c["op"] == "attention":
        _prepare_attention(c, s, g, r)
    else:
        _prepare_verify(c, s, g, r)
    return s


def _randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _cache(g, c, pages):
    """[pages, Hk, page size, D]; token-major in memory for layout "nhd"."""
    dt = TYPES[c["dtype"]]
    if c["layout"] == "nhd":
        return _randn(g, pages, c["ps"], c["Hk"], c["D"], dtype=dt).transpose(1, 2)
    return _randn(g, pages, c["Hk"], c["ps"], c["D"], dtype=dt)


def _prepare_append(c, s, g):
    T, D, dt = c["T"], c["D"], TYPES[c["dtype"]]
    pages = -(-T // c["ps"]) + 3
    s["qkv"] = _randn(g, T, (c["Hq"] + 2 * c["Hk"]) * D, dtype=dt)
    s["k_cache"], s["v_cache"] = _cache(g, c, pages), _cache(g, c, pages)
    # pages in any order, as an allocator hands them out; skipped tokens have the slot -1
    order = torch.randperm(pages, generator=g, device=DEV)
    t = torch.arange(T, device=DEV)
    s["slots"] = order[t // c["ps"]] * c["ps"] + t % c["ps"]
    if c["skip"] > 0:
        s["slots"][torch.randperm(T, generator=g, device=DEV)[: int(round(T * c["skip"]))]] = -1
    s["positions"] = (t + torch.randint(0, MAX_POS - T, (1,), generator=g, device=DEV)) % MAX_POS
    inv = THETA ** (-torch.arange(0, c["R"], 2, device=DEV, dtype=torch.float64) / c["R"])
    angle = torch.arange(MAX_POS, device=DEV, dtype=torch.float64)[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["q_weight"] = s["k_weight"] = None
    if c["norm"]:
        s["q_weight"] = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dt)
        s["k_weight"] = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dt)


def _prepare_attention(c, s, g, r):
    B, L, ps = c["B"], c["L"], c["ps"]
    n = _lengths(c)
    r.shuffle(n)
    need = [-(-v // ps) for v in n]
    pages, width = sum(need) + 2, max(max(need), 1)
    s["k_cache"], s["v_cache"] = _cache(g, c, pages), _cache(g, c, pages)
    s["q"] = _randn(g, B, L, c["Hq"], c["D"], dtype=TYPES[c["dtype"]], scale=2.0)
    s["seq_lens"] = torch.tensor(n, dtype=torch.int32, device=DEV)
    # each sequence's pages, in any order; the places after its last page are unused
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    counts = torch.tensor(need, device=DEV)
    at = (counts.cumsum(0) - counts)[:, None] + torch.arange(width, device=DEV)
    used = torch.arange(width, device=DEV) < counts[:, None]
    s["page_table"] = torch.where(used, order[at.clamp(max=pages - 1)], torch.full_like(at, -1, dtype=torch.int32))
    s["tail_mask"] = None
    if c["mask"] == "tail":
        # drafted rows see themselves and some of the others
        m = torch.rand(B, L, L, generator=g, device=DEV) < 0.6
        s["tail_mask"] = m | torch.eye(L, dtype=torch.bool, device=DEV)
    s["scale"] = c["D"] ** -0.5


def _prepare_verify(c, s, g, r):
    B, K, V, dt = c["B"], c["K"], c["V"], TYPES[c["dtype"]]

    def logits(rows):
        x = torch.randn(B, rows, V, generator=g, device=DEV) * 2.5
        # a few likely tokens in each row, as a trained head has
        return x.add_(12.0 * (torch.rand(B, rows, V, generator=g, device=DEV) < 6.0 / V))

    target = logits(K + 1)
    draft = target[:, :K] + torch.randn(B, K, V, generator=g, device=DEV) * 0.7
    s["temperature"] = None
    t = torch.ones(B, device=DEV)
    if c["temp"] == "mixed":   # a greedy sequence now and then
        t = torch.rand(B, generator=g, device=DEV) * 0.9 + 0.4
        t[torch.rand(B, generator=g, device=DEV) < 0.15] = 0.0
        s["temperature"] = t
    # drafted tokens: drawn from the draft's distribution at that temperature
    e = torch.empty(B, K, V, device=DEV).exponential_(generator=g)
    s["draft_tokens"] = (draft / t.clamp(min=0.05)[:, None, None] - e.log()).argmax(-1)
    s["target_logits"] = target.to(dt)
    s["draft_logits"] = draft.to(dt) if c["draft"] == "logits" else None
    s["uniform"] = torch.rand(B, K, generator=g, device=DEV)
    s["noise"] = torch.empty(B, V, device=DEV).exponential_(generator=g).clamp_(min=1e-20)
    s["n_draft"] = None
    if c["ragged"]:
        d = _draft_counts(c)
        r.shuffle(d)
        s["n_draft"] = torch.tensor(d, dtype=torch.int32, device=DEV)
        s["draft_tokens"].masked_fill_(torch.arange(K, device=DEV) >= s["n_draft"][:, None], -1)


# ------------------------------------------------------------------ one pass
_entries = None


def _framework():
    global _entries
    if _entries is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "simsd-release_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from kernels import paged_cache, spec_verify
        _entries = (paged_cache.paged_append, paged_cache.paged_attention, spec_verify.speculative_verify)
    return _entries


def run(s):
    with torch.inference_mode():
        if not own:
            return {"append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}[s["op"]](s)
        append, attention, verify = _framework()
        if s["op"] == "append":
            q = append(s["qkv"], s["Hq"], s["Hk"], s["k_cache"], s["v_cache"], s["slots"], s["positions"], s["cos"],
                       s["sin"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        if s["op"] == "attention":
            o, lse = attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["seq_lens"], scale=s["scale"],
                               tail_mask=s["tail_mask"], return_lse=True)
            return {"o": o, "lse": lse}
        tokens, accepted, logprobs = verify(s["target_logits"], s["draft_tokens"], s["uniform"], s["noise"],
                                            draft_logits=s["draft_logits"], temperature=s["temperature"],
                                            n_draft=s["n_draft"])
        return {"tokens": tokens, "accepted": accepted, "logprobs": logprobs}


def _plain_append(s):
    Hq, Hk, D, R, ps = s["Hq"], s["Hk"], s["D"], s["R"], s["ps"]
    x = s["qkv"].view(-1, Hq + 2 * Hk, D)
    qk = x[:, : Hq + Hk].float()
    if s["norm"]:
        w = torch.cat([s["q_weight"].float().expand(Hq, D), s["k_weight"].float().expand(Hk, D)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    a, b = qk[..., : R // 2], qk[..., R // 2: R]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin, qk[..., R:]], -1).to(x.dtype)
    kept = s["slots"] >= 0
    at = s["slots"][kept]
    s["k_cache"][at // ps, :, at % ps] = qk[kept, Hq:]
    s["v_cache"][at // ps, :, at % ps] = x[kept, Hq + Hk:]
    q = torch.where(kept[:, None, None], qk[:, :Hq], torch.zeros((), dtype=x.dtype, device=x.device))
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    q, n = s["q"], s["seq_lens"].long()
    B, L, Hq, D = q.shape
    Hk, ps = s["Hk"], s["ps"]
    G, width = Hq // Hk, s["page_table"].shape[1] * ps
    table = s["page_table"].long().clamp(min=0)
    j = torch.arange(width, device=q.device)
    stored = j < n[:, None]
    k = s["k_cache"][table].transpose(1, 2).reshape(B, Hk, width, D).float()
    v = s["v_cache"][table].transpose(1, 2).reshape(B, Hk, width, D).float().masked_fill_(~stored[:, None, :, None], 0.0)
    rows = q.view(B, L, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * L, D).float()
    score = (rows @ k.transpose(2, 3) * s["scale"]).view(B, Hk, G, L, width)
    tail = j - (n[:, None] - L)                                           # < 0: before the newest L keys
    t = torch.arange(L, device=q.device)
    if s["tail_mask"] is None:
        seen = tail[:, None] <= t[:, None]
    else:
        seen = (tail < 0)[:, None] | s["tail_mask"].gather(2, tail.clamp(0, L - 1)[:, None].expand(B, L, width))
    score = score.masked_fill(~(seen & stored[:, None])[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, G * L, width) @ v).view(B, Hk, G, L, D) / total.masked_fill(total == 0, 1.0)
    lse = (top + total.log()).squeeze(-1)
    return {"o": o.permute(0, 3, 1, 2, 4).reshape(B, L, Hq, D).to(q.dtype),
            "lse": lse.permute(0, 3, 1, 2).reshape(B, L, Hq)}


def _plain_distribution(logits, temperature):
    """(probabilities, log probabilities) over the last axis; greedy where the temperature is 0."""
    x = logits.float()
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=FLT_MAX)
    top = x.amax(-1, keepdim=True)
    z = x - top.masked_fill(top == -math.inf, 0.0)
    if temperature is not None:
        t = temperature.view(-1, 1, 1)
        first = torch.where(z == 0, torch.arange(x.shape[-1], device=x.device), x.shape[-1]).amin(-1, keepdim=True)
        greedy = torch.where(torch.arange(x.shape[-1], device=x.device) == first, 0.0, -math.inf)
        z = torch.where(t > 0, z / t.clamp(min=1e-30), greedy)
    w = torch.exp(z)
    total = w.sum(-1, keepdim=True)
    total = total.masked_fill(total == 0, 1.0)
    return w / total, z - total.log()


def _plain_verify(s):
    x, u, noise = s["draft_tokens"], s["uniform"], s["noise"]
    B, K = x.shape
    V = noise.shape[1]
    count = torch.full((B,), K, device=x.device) if s["n_draft"] is None else s["n_draft"].long()
    p, logp = _plain_distribution(s["target_logits"], s["temperature"])
    at = x.clamp(min=0)[:, :, None]
    q = torch.zeros_like(p).scatter_(2, torch.cat([at, at[:, :1]], 1), 1.0)
    if s["draft_logits"] is not None:
        q[:, :K] = _plain_distribution(s["draft_logits"], s["temperature"])[0]
    step = torch.arange(K, device=x.device)
    ok = u * q[:, :K].gather(2, at)[..., 0] < p[:, :K].gather(2, at)[..., 0]
    n = (ok & (step < count[:, None])).long().cumprod(1).sum(1)
    row = n[:, None, None].expand(B, 1, V)
    pr = p.gather(1, row)[:, 0]
    qr = torch.where((n < count)[:, None], q.gather(1, row)[:, 0], torch.zeros((), device=x.device))
    left = (pr - qr).clamp(min=0)
    left = torch.where(left.amax(1, keepdim=True) > 0, left, pr)           # p nowhere over q: drawn from p
    race = left / noise
    best = race == race.amax(1, keepdim=True)
    new = torch.where(best, torch.arange(V, device=x.device), V).amin(1, keepdim=True)
    place = torch.arange(K + 1, device=x.device)
    drafted = torch.cat([x, x[:, :1]], 1)
    tokens = torch.where(place < n[:, None], drafted, torch.where(place == n[:, None], new, -1))
    lp = logp.gather(2, tokens.clamp(min=0)[:, :, None])[..., 0]
    return {"tokens": tokens, "accepted": n, "logprobs": torch.where(tokens >= 0, lp, torch.zeros((), device=x.device))}


# ------------------------------------------------------------------ in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    return {"append": _exact_append, "attention": _exact_attention, "verify": _exact_verify}[c["op"]](s)


def _exact_append(s):
    Hq, Hk, D, R = s["Hq"], s["Hk"], s["D"], s["R"]
    x = s["qkv"].double().view(-1, Hq + 2 * Hk, D)
    turn = torch.complex(s["cos"][s["positions"]].double(), s["sin"][s["positions"]].double())

    def rotated(part, weight):
        if weight is not None:
            part = torch.nn.functional.normalize(part, dim=-1, eps=0.0) * math.sqrt(D) * _shrink(part) * weight.double()
        z = torch.complex(part[..., : R // 2], part[..., R // 2: R]) * turn[:, None]
        return torch.cat([z.real, z.imag, part[..., R:]], -1)

    def _shrink(part):   # |x| / sqrt(|x|^2 + D eps)
        sq = part.pow(2).sum(-1, keepdim=True)
        return (sq / (sq + D * EPS)).sqrt()

    q, k, v = rotated(x[:, :Hq], s["q_weight"]), rotated(x[:, Hq:Hq + Hk], s["k_weight"]), x[:, Hq + Hk:]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    for t, slot in enumerate(s["slots"].tolist()):
        if slot < 0:
            q[t] = 0
        else:
            kc[slot // s["ps"], :, slot % s["ps"]] = k[t]
            vc[slot // s["ps"], :, slot % s["ps"]] = v[t]
    return {"q": q, "k_cache": kc, "v_cache": vc}


def _exact_attention(s):
    q = s["q"].double()
    B, L, Hq, D = q.shape
    G = Hq // s["Hk"]
    o = torch.zeros_like(q)
    lse = torch.full((B, L, Hq), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(s["seq_lens"].tolist()):
        if n == 0:
            continue
        pages = s["page_table"][b, : -(-n // s["ps"])].long()
        for h in range(s["Hk"]):
            k = s["k_cache"][pages, h].reshape(-1, D)[:n].double()
            v = s["v_cache"][pages, h].reshape(-1, D)[:n].double()
            for t in range(L):
                see = torch.ones(n, dtype=torch.bool, device=q.device)
                for i in range(max(0, L - n), L):
                    see[n - L + i] = i <= t if s["tail_mask"] is None else s["tail_mask"][b, t, i]
                if not bool(see.any()):
                    continue
                z = (q[b, t, h * G:(h + 1) * G] @ k[see].T) * s["scale"]
                lse[b, t, h * G:(h + 1) * G] = torch.logsumexp(z, -1)
                o[b, t, h * G:(h + 1) * G] = torch.softmax(z, -1) @ v[see]
    return {"o": o, "lse": lse}


def _exact_verify(s):
    x, V = s["draft_tokens"].tolist(), s["noise"].shape[1]
    B, K = len(x), len(x[0])
    out = torch.zeros(B, K + 1, dtype=torch.float64, device=DEV)

    def law(row, t):
        row = row.double()
        return torch.log_softmax(row / t, -1) if t > 0 else torch.where(
            torch.arange(V, device=DEV) == int((row == row.max()).nonzero()[0]), 0.0, -math.inf).double()

    for b in range(B):
        t = 1.0 if s["temperature"] is None else float(s["temperature"][b])
        count = K if s["n_draft"] is None else int(s["n_draft"][b])
        i = 0
        while True:
            p = law(s["target_logits"][b, i], t)
            if i == count:
                left = p.exp()
            else:
                q = law(s["draft_logits"][b, i], t).exp() if s["draft_logits"] is not None else \
                    torch.nn.functional.one_hot(torch.tensor(x[b][i], device=DEV), V).double()
                if float(s["uniform"][b, i]) * float(q[x[b][i]]) < float(p[x[b][i]].exp()):
                    out[b, i] = p[x[b][i]]
                    i += 1
                    continue
                left = (p.exp() - q).clamp(min=0)
                left = left if float(left.max()) > 0 else p.exp()
            out[b, i] = p[int((left / s["noise"][b].double()).argmax())]
            break
    return {"tokens": None, "accepted": None, "logprobs": out}
