"""Measured cases of the serving operators around the paged cache: the cache held in
8 bits, attention through a window, the page tables, and the rules on logits.

* ``append``: q/k RMSNorm and rotary embedding of the merged q/k/v projection, keys and
  values written in 8 bits (e4m3) with a scale for each block of tokens and head
  (`paged_append8`).
* ``attention``: attention of the newest token, or of a few drafted ones, over the
  8-bit cache (`paged_attention8`); through a sliding window that leaves a few first
  tokens visible, over the 8-bit or the 16-bit cache (`paged_attention`).
* ``reserve``: pages for each sequence's next tokens, their slots and positions, and the
  way back for tokens that were not kept (`paged_reserve`, `paged_release`).
* ``rules``: penalties for repeated tokens, biases and grammar masks on the target's
  logits of every drafted row (`adjust_logits`).

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
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
EPS = 1e-6
THETA = 1e6


# ------------------------------------------------------------------ the cases
def listed():
    """8B-shaped heads (32 query, 8 key-value, 128 wide) where nothing else is said."""
    return [
        # one sequence's next four drafted tokens, in the middle of a block: all latency
        _append("append8-1x4", B=1, L=4),
        # a long prompt chunk of four sequences, some rows padding
        _append("append8-4x2048", B=4, L=2048, pad=0.3),
        # one short conversation, one new token: the smallest read, all latency
        _attention("attend8-1x100", B=1, L=1, lo=100, hi=100),
        # an ordinary serving batch, ragged, one new token each
        _attention("attend8-32x2k", B=32, L=1, lo=300, hi=4096),
        # two long documents: the cache's length has to be split over the whole GPU
        _attention("attend8-2x128k", B=2, L=1, lo=120000, hi=131072, ps=64, block=64),
        # verification of 8 drafted rows per sequence under a block mask
        _attention("attend8-verify-16x8", B=16, L=8, lo=1000, hi=3000, mask="tail"),
        # long chats through a window, 16-bit cache, a few first tokens kept
        _attention("window-16x32k", B=16, L=1, lo=8000, hi=32768, bits=16, window=4096, sinks=4),
        # verification of 5 drafted rows through a short window, 8-bit token-major cache, odd sizes
        _attention("window8-verify-19x5", B=19, L=5, lo=1, hi=9000, Hq=28, Hk=4, window=1000, sinks=70, ps=24, block=8,
                   layout="nhd", dtype="fp16"),
        # a decoding batch's next four places
        _reserve("reserve-32x4", B=32, L=4, lo=100, hi=4096),
        # prompts of a new batch, ragged
        _reserve("reserve-prompts-64x2k", B=64, L=2048, lo=0, hi=0),
        # one sequence's next token, a small odd vocabulary, 32-bit logits
        _rules("rules-1x1-odd", B=1, K=0, V=50021, dtype="fp32"),
        # a large batch of drafted rows over the 8B model's vocabulary
        _rules("rules-64x8", B=64, K=7, V=151936),
    ]


def _append(name=None, **kw):
    return _case(name, dict(op="append", B=1, L=1, Hq=32, Hk=8, D=128, R=kw.get("D", 128), ps=16, block=16, norm=True,
                            dtype="bf16", layout="hnd", pad=0.0, back=1000), kw)


def _attention(name=None, **kw):
    return _case(name, dict(op="attention", B=1, L=1, lo=1, hi=1, Hq=32, Hk=8, D=128, ps=16, block=16, bits=8, window=0,
                            sinks=0, pow2=True, dtype="bf16", layout="hnd", mask="causal", empty=0.0), kw)


def _reserve(name=None, **kw):
    return _case(name, dict(op="reserve", B=1, L=1, lo=0, hi=0, ps=16, short=False), kw)


def _rules(name=None, **kw):
    return _case(name, dict(op="rules", B=1, K=0, V=1, dtype="bf16", penalties=True, seen=True, bias=300, mask="rows"), kw)


def _case(name, base, kw):
    base.update(kw)
    if name is not None:
        base["name"] = name
    return base


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "window", "reserve", "rules"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "reserve":
        L = _log_int(rng, 1, 2048)
        hi = rng.choice([0, _log_int(rng, 1, 30000)])
        return _reserve(B=_log_int(rng, 1, min(512, max(1, 131072 // L))), L=L, lo=rng.randint(0, hi), hi=hi,
                        ps=rng.choice([1, 8, 16, 16, 24, 64, 128]), short=rng.random() < 0.2)
    if op == "rules":
        V = rng.choice([151936, 32000, _log_int(rng, 1000, 151936)])
        K = rng.randint(0, 8)
        return _rules(B=_log_int(rng, 1, max(1, min(64, 64 * 8 * 151936 // (V * (K + 1) * 2)))), K=K, V=V,
                      dtype=rng.choice([dtype, "fp32"]), penalties=rng.random() < 0.8, seen=rng.random() < 0.6,
                      bias=rng.choice([0, 1, 30, 300]), mask=rng.choice(["none", "sequences", "rows"]))
    D = rng.choice([128, 128, 64])
    Hk = rng.choice([1, 2, 4, 8, 8])
    Hq = Hk * rng.choice([1, 2, 4, 4, 5, 7, 8])
    ps = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    block = rng.choice([b for b in (1, 2, 4, 8, 16, 24, 32, 64) if ps % b == 0])
    layout = rng.choice(["hnd", "nhd"])
    if op == "append":
        L = _log_int(rng, 1, 2048)
        most = (8192 if Hq + 2 * Hk <= 48 else 4096) // L
        return _append(B=_log_int(rng, 1, max(1, min(64, most))), L=L, Hq=Hq, Hk=Hk, D=D, R=rng.choice([D, D, D // 2]), ps=ps,
                       block=block, norm=rng.random() < 0.7, dtype=dtype, layout=layout, pad=rng.choice([0.0, 0.3]),
                       back=rng.choice([0, 1000]))
    B = _log_int(rng, 1, 128)
    hi = _log_int(rng, 8, max(8, min(131072, (1 << 28) // (B * Hk * D))))
    c = dict(B=B, L=rng.choice([1, 1, 1, 2, 4, 5, 8, 16]), lo=_log_int(rng, 1, hi), hi=hi, Hq=Hq, Hk=Hk, D=D, ps=ps,
             block=block, dtype=dtype, layout=layout, mask=rng.choice(["causal", "tail"]), empty=rng.choice([0.0, 0.1]),
             pow2=rng.random() < 0.6)
    if op == "window":
        c.update(bits=rng.choice([8, 16]), window=_log_int(rng, 1, hi), sinks=rng.choice([0, 1, 4, 64, 100]))
    return _attention(**c)


def _lengths(c):
    """The case's lengths: the same multiset for every seed, so that its work is the case's own."""
    r = random.Random(c["B"] * 7919 + c["hi"])
    n = [_log_int(r, max(1, c["lo"]), max(1, c["hi"])) if c["hi"] > 0 else 0 for _ in range(c["B"])]
    n[0] = c["hi"]
    return [0 if i > 0 and r.random() < c.get("empty", 0.0) else v for i, v in enumerate(n)]


def _new_counts(c):
    """(new tokens, length after them) of each sequence: all L are new, or fewer where the case has padding."""
    r = random.Random(c["B"] * 31 + c["L"])
    new = [r.randint(0, c["L"]) if i > 0 and r.random() < c["pad"] else c["L"] for i in range(c["B"])]
    return [(v, v + r.randint(0, c["back"])) for v in new]


def _prompt_counts(c):
    r = random.Random(c["B"] * 17 + c["L"])
    return [c["L"]] + [r.randint(0, c["L"]) if c["L"] > 16 else c["L"] for _ in range(c["B"] - 1)]


def _seen_keys(c, n):
    """Keys of a sequence of n that some query sees."""
    if not c["window"]:
        return n
    first = max(0, n - c["L"] + 1 - c["window"])
    return n - first + min(c["sinks"], first)


def work(c):
    e = 4 if c.get("dtype") == "fp32" else 2
    if c["op"] == "append":
        T, D, H = sum(v for v, _ in _new_counts(c)), c["D"], c["Hq"] + 2 * c["Hk"]
        # the projections read, q and the new keys and values written, their blocks' scales, one table row a token
        return {"bytes": T * (H * D * e + c["Hq"] * D * e + 2 * c["Hk"] * D + c["R"] * 4) + T * 2 * c["Hk"] * 4 // c["block"]
                + c["B"] * 8, "flops": T * ((c["Hq"] + c["Hk"]) * (3 * c["R"] + 4 * D) + 2 * c["Hk"] * 3 * D)}
    if c["op"] == "attention":
        n = [_seen_keys(c, v) for v in _lengths(c)]
        a_key = 2 * c["D"] * 2 if c["bits"] == 16 else 2 * c["D"] + 8 / c["block"]
        qo = c["B"] * c["L"] * c["Hq"] * (2 * c["D"] * e + 4)
        pages = sum(-(-v // c["ps"]) for v in n) * 4
        return {"bytes": sum(n) * c["Hk"] * a_key + qo + pages, "flops": 4 * sum(n) * c["L"] * c["Hq"] * c["D"]}
    if c["op"] == "reserve":
        new = _prompt_counts(c)
        pages = sum(new) // c["ps"]
        return {"bytes": c["B"] * (c["L"] * 16 + 28) + pages * 16, "flops": c["B"] * c["L"] * 4}
    rows = c["B"] * (c["K"] + 1)
    masks = {"none": 0, "sequences": c["B"], "rows": rows}[c["mask"]]
    return {"bytes": rows * c["V"] * 2 * e + c["B"] * c["V"] * (4 if c["penalties"] else 0)
            + (masks + (c["B"] if c["seen"] and c["penalties"] else 0)) * c["V"] // 8, "flops": 6 * rows * c["V"]}


# ------------------------------------------------------------------ inputs
def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    r = random.Random(int(seed))
    s = dict(c)
    s.pop("name", None)
    {"append": _prepare_append, "attention": _prepare_attention, "reserve": _prepare_reserve, "rules": _prepare_rules}[
        c["op"]](c, s, g, r)
    return s


def _randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _cache(g, c, pages):
    """[pages, Hk, page size, D]; token-major in memory for layout "nhd"."""
    dt = TYPES[c["dtype"]]
    if c["layout"] == "nhd":
        return _randn(g, pages, c["ps"], c["Hk"], c["D"], dtype=dt).transpose(1, 2)
    return _randn(g, pages, c["Hk"], c["ps"], c["D"], dtype=dt)


def _cache8(g, c, pages):
    """An 8-bit cache and its scales [pages, Hk, page size / block]: blocks of different magnitudes."""
    n = c["ps"] // c["block"]
    x = torch.randn(pages, c["Hk"], n, c["block"], c["D"], generator=g, device=DEV)
    x *= torch.exp(0.7 * torch.randn(pages, c["Hk"], n, 1, 1, generator=g, device=DEV))
    top = x.abs().amax((-1, -2))
    scale = _power(top) if c.get("pow2", True) else top / F8_MAX
    x = (x / scale[..., None, None]).clamp_(-F8_MAX, F8_MAX).to(F8).view(pages, c["Hk"], c["ps"], c["D"])
    if c["layout"] == "nhd":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    return x, scale.contiguous()


def _power(top):
    """The smallest power of two s, 2^-64 to 2^64, with top <= 448 s."""
    m, e = torch.frexp(top)
    e = torch.where(m <= F8_MAX / 512, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(top), torch.where(top > 0, e, -64).clamp(-64, 64))


def _tables(g, c, need, spare=2):
    """Page tables of sequences that need so many pages: pages in any order, unused places -1."""
    pages, width = sum(need) + spare, max(max(need), 1)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    counts = torch.tensor(need, device=DEV)
    at = (counts.cumsum(0) - counts)[:, None] + torch.arange(width, device=DEV)
    used = torch.arange(width, device=DEV) < counts[:, None]
    return pages, torch.where(used, order[at.clamp(max=pages - 1)], torch.full_like(at, -1, dtype=torch.int32))


def _prepare_append(c, s, g, r):
    B, L, D, dt = c["B"], c["L"], c["D"], TYPES[c["dtype"]]
    both = _new_counts(c)
    r.shuffle(both)
    new, total = [v for v, _ in both], [v for _, v in both]
    pages, s["page_table"] = _tables(g, c, [-(-v // c["ps"]) for v in total])
    s["qkv"] = _randn(g, B, L, (c["Hq"] + 2 * c["Hk"]) * D, dtype=dt)
    s["k_cache"], s["k_scale"] = _cache8(g, c, pages)
    s["v_cache"], s["v_scale"] = _cache8(g, c, pages)
    s["seq_lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
    s["count"] = torch.tensor(new, dtype=torch.int32, device=DEV) if c["pad"] > 0 else None
    inv = THETA ** (-torch.arange(0, c["R"], 2, device=DEV, dtype=torch.float64) / c["R"])
    angle = torch.arange(max(max(total), 1), device=DEV, dtype=torch.float64)[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["q_weight"] = s["k_weight"] = None
    if c["norm"]:
        s["q_weight"] = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dt)
        s["k_weight"] = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dt)


def _prepare_attention(c, s, g, r):
    B, L = c["B"], c["L"]
    n = _lengths(c)
    r.shuffle(n)
    pages, s["page_table"] = _tables(g, c, [-(-v // c["ps"]) for v in n])
    if c["bits"] == 8:
        s["k_cache"], s["k_scale"] = _cache8(g, c, pages)
        s["v_cache"], s["v_scale"] = _cache8(g, c, pages)
    else:
        s["k_cache"], s["v_cache"] = _cache(g, c, pages), _cache(g, c, pages)
    s["q"] = _randn(g, B, L, c["Hq"], c["D"], dtype=TYPES[c["dtype"]], scale=2.0)
    s["seq_lens"] = torch.tensor(n, dtype=torch.int32, device=DEV)
    s["tail_mask"] = None
    if c["mask"] == "tail":
        # drafted rows see themselves and some of the others
        m = torch.rand(B, L, L, generator=g, device=DEV) < 0.6
        s["tail_mask"] = m | torch.eye(L, dtype=torch.bool, device=DEV)
    s["scale"] = c["D"] ** -0.5


def _prepare_reserve(c, s, g, r):
    both = list(zip(_lengths(c), _prompt_counts(c)))
    r.shuffle(both)
    n, new = [v for v, _ in both], [v for _, v in both]
    held = [-(-v // c["ps"]) for v in n]
    most = -(-(c["hi"] + c["L"]) // c["ps"])
    wanted = sum(-(-(a + b) // c["ps"]) - h for a, b, h in zip(n, new, held))
    spare = wanted // 2 if c["short"] else wanted + 7   # a pool that does not go round now and then
    pages, table = _tables(g, c, held, spare=max(spare, 1))
    s["page_table"] = torch.full((c["B"], most), -1, dtype=torch.int32, device=DEV)
    s["page_table"][:, : min(table.shape[1], most)] = table[:, :most]
    used = torch.zeros(pages, dtype=torch.bool, device=DEV)
    used[table[table >= 0].long()] = True
    free = (~used).nonzero()[:, 0].to(torch.int32)
    free = free[torch.randperm(free.numel(), generator=g, device=DEV)]
    s["free_pages"] = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    s["free_pages"][: free.numel()] = free
    s["free_count"] = torch.tensor([free.numel()], dtype=torch.int32, device=DEV)
    s["lens"] = torch.tensor(n, dtype=torch.int32, device=DEV)
    s["held"] = torch.tensor(held, dtype=torch.int32, device=DEV)
    s["count"] = torch.tensor(new, dtype=torch.int32, device=DEV)


def _prepare_rules(c, s, g, r):
    B, K, V, R = c["B"], c["K"], c["V"], c["K"] + 1
    x = torch.randn(B, R, V, generator=g, device=DEV) * 2.5
    s["logits"] = x.add_(12.0 * (torch.rand(B, R, V, generator=g, device=DEV) < 6.0 / V)).to(TYPES[c["dtype"]])
    s["drafts"] = torch.randint(0, V, (B, K), generator=g, device=DEV)
    s["counts"] = s["seen"] = s["repetition"] = s["presence"] = s["frequency"] = None
    words = -(-V // 32)
    if c["penalties"]:
        # some hundreds of answered tokens, a few of them many times
        s["counts"] = torch.zeros(B, V, dtype=torch.int32, device=DEV)
        at = (torch.rand(B, 600, generator=g, device=DEV) ** 3 * V).long().clamp_(max=V - 1)
        s["counts"].scatter_add_(1, at, torch.ones_like(at, dtype=torch.int32))
        if K > 1:   # a drafted token that was answered before, and one drafted twice
            s["drafts"][:, 0] = at[:, 0]
            s["drafts"][:, 1] = at[:, 0]
        s["repetition"] = torch.rand(B, generator=g, device=DEV) * 0.5 + 1.0
        s["presence"] = torch.rand(B, generator=g, device=DEV)
        s["frequency"] = torch.rand(B, generator=g, device=DEV) * 0.5
        if c["seen"]:   # tokens of the prompt
            s["seen"] = _words(torch.rand(B, words * 32, generator=g, device=DEV) < 0.01)
    s["bias_ids"] = s["bias_values"] = None
    if c["bias"] > 0:
        ids = torch.rand(B, c["bias"], generator=g, device=DEV) * V
        s["bias_ids"] = ids.to(torch.int32).clamp_(max=V - 1)
        s["bias_ids"][torch.rand(B, c["bias"], generator=g, device=DEV) < 0.2] = -1   # shorter lists
        s["bias_values"] = torch.randn(B, c["bias"], generator=g, device=DEV) * 5.0
    s["allowed"] = None
    if c["mask"] != "none":
        # half the sequences follow a grammar that leaves few tokens, the others are free
        rows = B * (R if c["mask"] == "rows" else 1)
        few = torch.rand(rows, words * 32, generator=g, device=DEV) < 0.02
        free = torch.rand(rows, 1, generator=g, device=DEV) < 0.5
        s["allowed"] = _words(few | free).view(*((B, R) if c["mask"] == "rows" else (B,)), words)


def _words(bits):
    """[.., 32 n] truth values as [.., n] int32, token v in bit v % 32 of word v / 32."""
    w = bits.view(*bits.shape[:-1], -1, 32).long() << torch.arange(32, device=DEV)
    w = w.sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


# ------------------------------------------------------------------ one pass
_entries = None


def _framework():
    global _entries
    if _entries is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "simsd-release_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from kernels import logit_rules, paged_cache, paged_cache8, paged_tables
        _entries = (paged_cache8.paged_append8, paged_cache8.paged_attention8, paged_cache.paged_attention,
                    paged_tables.paged_reserve, paged_tables.paged_release, logit_rules.adjust_logits)
    return _entries


def run(s):
    with torch.inference_mode():
        if not own:
            return {"append": _plain_append, "attention": _plain_attention, "reserve": _plain_reserve, "rules": _plain_rules}[
                s["op"]](s)
        append, attention8, attention, reserve, release, adjust = _framework()
        if s["op"] == "append":
            q = append(s["qkv"], s["Hq"], s["Hk"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["page_table"],
                       s["seq_lens"], s["cos"], s["sin"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS,
                       count=s["count"])
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if s["op"] == "attention":
            more = dict(scale=s["scale"], tail_mask=s["tail_mask"], return_lse=True, window=s["window"] or None,
                        sinks=s["sinks"])
            if s["bits"] == 8:
                o, lse = attention8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["page_table"],
                                    s["seq_lens"], **more)
            else:
                o, lse = attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["seq_lens"], **more)
            return {"o": o, "lse": lse}
        if s["op"] == "reserve":
            slots, positions, total = reserve(s["page_table"], s["lens"], s["held"], s["free_pages"], s["free_count"], s["L"],
                                              s["ps"], count=s["count"])
            # none of the tokens was kept: their pages go back
            release(s["page_table"], s["held"], s["free_pages"], s["free_count"], s["lens"], s["ps"])
            return _pool(s, slots, positions, total)
        return {"logits": adjust(s["logits"], counts=s["counts"], drafts=s["drafts"], repetition=s["repetition"],
                                 presence=s["presence"], frequency=s["frequency"], seen=s["seen"], bias_ids=s["bias_ids"],
                                 bias_values=s["bias_values"], allowed=s["allowed"])}


def _pool(s, slots, positions, total):
    return {"slots": slots, "positions": positions, "total": total, "page_table": s["page_table"], "held": s["held"],
            "free_pages": s["free_pages"], "free_count": s["free_count"]}


def _plain_append(s):
    Hq, Hk, D, R, ps, bs = s["Hq"], s["Hk"], s["D"], s["R"], s["ps"], s["block"]
    B, L = s["qkv"].shape[:2]
    x = s["qkv"].view(B, L, Hq + 2 * Hk, D)
    qk = x[:, :, : Hq + Hk].float()
    if s["norm"]:
        w = torch.cat([s["q_weight"].float().expand(Hq, D), s["k_weight"].float().expand(Hk, D)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    total = s["seq_lens"].long()
    new = torch.full_like(total, L) if s["count"] is None else s["count"].long()
    t = torch.arange(L, device=x.device)
    pos = total[:, None] - L + t
    real = (t >= L - new[:, None]) & (pos >= 0)
    at = pos.clamp(min=0)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    a, b = qk[..., : R // 2], qk[..., R // 2: R]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin, qk[..., R:]], -1)
    q = torch.where(real[:, :, None, None], qk[:, :, :Hq], torch.zeros((), device=x.device)).to(x.dtype)
    place = s["page_table"].gather(1, at // ps).long()[real] * ps + (at % ps)[real]        # slots of the new tokens
    # what is already in the block that the first new token goes to
    first = (total - new).clamp(min=0)
    j = torch.arange(bs, device=x.device)
    before = (first // bs * bs)[:, None] + j
    has = (before < first[:, None]) & (new > 0)[:, None]
    before = before.clamp(max=s["page_table"].shape[1] * ps - 1)
    older = s["page_table"].gather(1, before // ps).long()[has] * ps + (before % ps)[has]
    blocks = s["k_scale"].shape[0] * (ps // bs)
    fresh = torch.zeros(blocks, dtype=torch.bool, device=x.device)
    fresh[place[place % bs == 0] // bs] = True
    for cache, scale, y in ((s["k_cache"], s["k_scale"], qk[:, :, Hq:][real]), (s["v_cache"], s["v_scale"], x[:, :, Hq + Hk:][real].float())):
        top = torch.zeros(blocks, Hk, device=x.device)
        top.scatter_reduce_(0, (place // bs)[:, None].expand(-1, Hk), y.abs().masked_fill(~y.isfinite(), 0.0).amax(-1), "amax")
        old = scale.transpose(1, 2).reshape(blocks, Hk)
        now = old.clone()
        at = place // bs
        now[at] = torch.where(fresh[at][:, None], _power(top)[at], torch.maximum(_power(top)[at], old[at]))
        bytes_ = cache.view(torch.uint8)
        was = bytes_[older // ps, :, older % ps].view(F8).float()
        was = _quantised(was * old[older // bs][..., None], now[older // bs][..., None])
        bytes_[older // ps, :, older % ps] = was.view(torch.uint8)
        bytes_[place // ps, :, place % ps] = _quantised(y, now[at][..., None]).view(torch.uint8)
        scale.copy_(now.view(scale.shape[0], -1, Hk).transpose(1, 2))
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _quantised(x, scale):
    y = (x / scale).clamp(-F8_MAX, F8_MAX)
    return torch.where(x.isfinite(), y, math.nan).to(F8)


def _plain_attention(s):
    q, n = s["q"], s["seq_lens"].long()
    B, L, Hq, D = q.shape
    Hk, ps = s["Hk"], s["ps"]
    G, width = Hq // Hk, s["page_table"].shape[1] * ps
    table = s["page_table"].long().clamp(min=0)
    j = torch.arange(width, device=q.device)
    stored = j < n[:, None]

    def whole(cache, scale):
        if s["bits"] == 16:
            return cache[table].transpose(1, 2).reshape(B, Hk, width, D).float()
        x = cache.view(torch.uint8)[table].view(F8).float()                            # [B, pages, Hk, ps, D]
        x = x.reshape(*x.shape[:3], ps // s["block"], s["block"], D) * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(B, Hk, width, D)

    k = whole(s["k_cache"], s.get("k_scale"))
    v = whole(s["v_cache"], s.get("v_scale")).masked_fill_(~stored[:, None, :, None], 0.0)
    rows = q.view(B, L, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * L, D).float()
    score = (rows @ k.transpose(2, 3) * s["scale"]).view(B, Hk, G, L, width)
    del k
    tail = j - (n[:, None] - L)                                           # < 0: before the newest L keys
    t = torch.arange(L, device=q.device)
    if s["tail_mask"] is None:
        seen = tail[:, None] <= t[:, None]
    else:
        seen = (tail < 0)[:, None] | s["tail_mask"].gather(2, tail.clamp(0, L - 1)[:, None].expand(B, L, width))
    if s["window"]:
        seen = seen & ((tail[:, None] > t[:, None] - s["window"]) | (j < s["sinks"]))
    score = score.masked_fill(~(seen & stored[:, None])[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, G * L, width) @ v).view(B, Hk, G, L, D) / total.masked_fill(total == 0, 1.0)
    lse = (top + total.log()).squeeze(-1)
    return {"o": o.permute(0, 3, 1, 2, 4).reshape(B, L, Hq, D).to(q.dtype),
            "lse": lse.permute(0, 3, 1, 2).reshape(B, L, Hq)}


def _plain_reserve(s):
    L, ps, table = s["L"], s["ps"], s["page_table"]
    lens, new = s["lens"].long(), s["count"].long()
    have = torch.maximum(s["held"].long(), (lens + ps - 1) // ps)
    need = torch.maximum((lens + new + ps - 1) // ps, have)
    take = need - have
    free = s["free_count"].long()
    fits = (take == 0) | (take.cumsum(0) <= free)
    given = torch.where(fits, new, 0)
    take = torch.where(fits, take, 0)
    start = take.cumsum(0) - take
    place = torch.arange(table.shape[1], device=table.device)
    order = place - have[:, None]                                          # of the sequence's new pages
    mine = (order >= 0) & (order < take[:, None])
    at = (free - 1 - start[:, None] - order).clamp(0, s["free_pages"].numel() - 1)
    table.copy_(torch.where(mine, s["free_pages"][at], table))
    s["held"].copy_(have + take)
    s["free_count"].sub_(take.sum().to(torch.int32))
    t = torch.arange(L, device=table.device)
    real = t >= L - given[:, None]
    positions = torch.where(real, (lens + given)[:, None] - L + t, 0)
    slots = torch.where(real, table.gather(1, positions // ps).long() * ps + positions % ps, -1)
    total = (lens + given).to(torch.int32)
    # back: the pages past those of `lens` tokens, sequence by sequence
    keep = torch.minimum((lens + ps - 1) // ps, s["held"].long())
    back = s["held"].long() - keep
    start = back.cumsum(0) - back + s["free_count"].long()
    order = place - keep[:, None]
    mine = (order >= 0) & (order < back[:, None])
    s["free_pages"].index_put_(((start[:, None] + order)[mine],), table[mine])
    s["free_count"].add_(back.sum().to(torch.int32))
    s["held"].copy_(keep)
    return _pool(s, slots, positions, total)


def _plain_bits(words, V):
    v = torch.arange(V, device=words.device)
    return (words[..., v >> 5] >> (v & 31) & 1).bool()


def _plain_rules(s):
    x = s["logits"].float()
    B, R, V = x.shape
    if s["counts"] is not None:
        drafted = torch.zeros(B, R, V, dtype=torch.int32, device=x.device)
        if R > 1:
            drafted[:, 1:].scatter_(2, s["drafts"][:, :, None], 1)
        c = s["counts"][:, None] + drafted.cumsum(1, dtype=torch.int32)
        met = c > 0
        again = met if s["seen"] is None else met | _plain_bits(s["seen"], V)[:, None]
        r = s["repetition"][:, None, None]
        x = torch.where(again, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None, None] * c - s["presence"][:, None, None] * met
    if s["bias_ids"] is not None:
        ids = s["bias_ids"].long()
        bias = torch.zeros(B, V + 1, dtype=torch.float64, device=x.device)
        bias.scatter_add_(1, torch.where(ids < 0, V, ids), s["bias_values"].double())
        x = x + bias[:, None, :V].float()
    if s["allowed"] is not None:
        ok = _plain_bits(s["allowed"], V)
        x = x.masked_fill(~(ok if ok.ndim == 3 else ok[:, None]), -math.inf)
    return {"logits": x.to(s["logits"].dtype)}


# ------------------------------------------------------------------ in 64 bits
def exact(c, seed):
    if c["op"] == "reserve":
        return None
    s = prepare(c, seed)
    return {"append": _exact_append, "attention": _exact_attention, "rules": _exact_rules}[c["op"]](s)


def _exact_append(s):
    """Stored values in units of their scales, not rounded to 8 bits."""
    Hq, Hk, D, R, ps, bs = s["Hq"], s["Hk"], s["D"], s["R"], s["ps"], s["block"]
    B, L = s["qkv"].shape[:2]
    x = s["qkv"].double().view(B, L, Hq + 2 * Hk, D)

    def rotated(part, weight, pos):
        if weight is not None:
            sq = part.pow(2).sum(-1, keepdim=True)
            part = part * (D / (sq + D * EPS)).sqrt() * weight.double()
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())
        z = torch.complex(part[..., : R // 2], part[..., R // 2: R]) * turn[:, None]
        return torch.cat([z.real, z.imag, part[..., R:]], -1)

    q = torch.zeros(B, L, Hq, D, dtype=torch.float64, device=DEV)
    caches = [s["k_cache"].view(torch.uint8).contiguous().view(F8).double(), s["v_cache"].view(torch.uint8).contiguous().view(F8).double()]
    scales = [s["k_scale"].double(), s["v_scale"].double()]
    for b, n in enumerate(s["seq_lens"].tolist()):
        new = min(n, L if s["count"] is None else int(s["count"][b]))
        if new == 0:
            continue
        pos = torch.arange(n - new, n, device=DEV)
        q[b, L - new:] = rotated(x[b, L - new:, :Hq], s["q_weight"], pos)
        table = s["page_table"][b].tolist()
        for cache, scale, y in zip(caches, scales, (rotated(x[b, L - new:, Hq:Hq + Hk], s["k_weight"], pos), x[b, L - new:, Hq + Hk:])):
            for lo in range((n - new) // bs * bs, n, bs):
                page, at, part = table[lo // ps], lo % ps, y[max(0, lo - (n - new)): lo + bs - (n - new)]
                i = max(0, n - new - lo)                                   # tokens of the block that were there
                want = part.abs().amax((0, 2)) / F8_MAX
                want = torch.exp2(torch.ceil(torch.log2(want)))
                old = scale[page, :, at // bs].clone()
                scale[page, :, at // bs] = want if i == 0 else torch.maximum(want, old)
                now = scale[page, :, at // bs]
                cache[page, :, at: at + i] *= (old / now)[:, None, None]
                cache[page, :, at + i: at + i + len(part)] = part.transpose(0, 1) / now[:, None, None]
    return {"q": q, "k_cache": caches[0], "v_cache": caches[1], "k_scale": scales[0], "v_scale": scales[1]}


def _exact_attention(s):
    q = s["q"].double()
    B, L, Hq, D = q.shape
    G = Hq // s["Hk"]
    o = torch.zeros_like(q)
    lse = torch.full((B, L, Hq), -math.inf, dtype=torch.float64, device=q.device)

    def values(name, pages, h, n):
        if s["bits"] == 16:
            return s[name + "_cache"][pages, h].reshape(-1, D)[:n].double()
        x = s[name + "_cache"].view(torch.uint8)[pages, h].view(F8).double()
        return (x * s[name + "_scale"][pages, h].double().repeat_interleave(s["block"], -1)[..., None]).reshape(-1, D)[:n]

    for b, n in enumerate(s["seq_lens"].tolist()):
        if n == 0:
            continue
        pages = s["page_table"][b, : -(-n // s["ps"])].long()
        j = torch.arange(n, device=q.device)
        for h in range(s["Hk"]):
            k, v = values("k", pages, h, n), values("v", pages, h, n)
            for t in range(L):
                see = torch.ones(n, dtype=torch.bool, device=q.device)
                for i in range(max(0, L - n), L):
                    see[n - L + i] = i <= t if s["tail_mask"] is None else s["tail_mask"][b, t, i]
                if s["window"]:
                    see &= (j + s["window"] > n - L + t) | (j < s["sinks"])
                if not bool(see.any()):
                    continue
                z = (q[b, t, h * G:(h + 1) * G] @ k[see].T) * s["scale"]
                lse[b, t, h * G:(h + 1) * G] = torch.logsumexp(z, -1)
                o[b, t, h * G:(h + 1) * G] = torch.softmax(z, -1) @ v[see]
    return {"o": o, "lse": lse}


def _exact_rules(s):
    x = s["logits"].double()
    B, R, V = x.shape
    for b in range(B):
        bias = torch.zeros(V, dtype=torch.float64, device=DEV)
        if s["bias_ids"] is not None:
            used = s["bias_ids"][b] >= 0
            bias.index_add_(0, s["bias_ids"][b][used].long(), s["bias_values"][b][used].double())
        count = None if s["counts"] is None else s["counts"][b].double()
        for i in range(R):
            y = x[b, i]
            if count is not None:
                if i > 0:
                    count[s["drafts"][b, i - 1]] += 1
                met = (count > 0).double()
                again = count > 0
                if s["seen"] is not None:
                    again = again | ((s["seen"][b].long()[:, None] >> torch.arange(32, device=DEV)) % 2 == 1).view(-1)[:V]
                factor = torch.where(y > 0, 1 / s["repetition"][b].double(), s["repetition"][b].double())
                y = y * torch.where(again, factor, 1.0) - s["frequency"][b].double() * count - s["presence"][b].double() * met
            y = y + bias
            if s["allowed"] is not None:
                words = s["allowed"][b] if s["allowed"].ndim == 2 else s["allowed"][b, i]
                ok = ((words.long()[:, None] >> torch.arange(32, device=DEV)) % 2 == 1).view(-1)[:V]
                y = torch.where(ok, y, -math.inf)
            x[b, i] = y
    return {"logits": x}
