"""What is timed when the operators of a long context in 8 bits are timed: rotary positions, the store into a cache of 8-bit codes
with a scale for each block of slots and KV head, the attention that reads it, and the eviction that keeps it at a budget.

Four kinds of case, by `op`:

    rope        queries and keys of T tokens rotated to their positions (`halves`: pairs (i, i + n_rot/2), else (2i, 2i + 1)), the
                first n_rot dimensions of each head, `scale` > 1: stretched to that many times the original context (YaRN)
    store       keys and values of up to `new` tokens for each of n sequences into the cache, and the touched blocks read back as
                the values that they stand for
    attention   up to `new` queries for each of n sequences of up to `kv` slots; `weights`: the probabilities are added up per slot
    evict       n sequences of up to `kv` slots cut to `keep` by their weights, and the kept slots read back as values

A cache is int8 [n, n_head_kv, n_ctx, hd] with scales float32 [n, n_head_kv, n_ctx / block].  The new tokens of a sequence are
rows q_start[i] .. q_start[i+1] of q / k / v, in slots pos0[i] and on.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16}
BASE, ORIG_CTX = 10000.0, 2048


def _rope(x, T, n_head, n_head_kv, hd, n_rot, halves, far, scale):
    return dict(op="rope", x=x, T=T, n_head=n_head, n_head_kv=n_head_kv, hd=hd, n_rot=n_rot, halves=halves, far=far, scale=scale)


def _store(x, n, new, n_head_kv, hd, n_ctx, block):
    return dict(op="store", x=x, n=n, new=new, n_head_kv=n_head_kv, hd=hd, n_ctx=n_ctx, block=block)


def _attention(x, n, new, n_head, n_head_kv, hd, kv, block, weights):
    return dict(op="attention", x=x, n=n, new=new, n_head=n_head, n_head_kv=n_head_kv, hd=hd, kv=kv, block=block, weights=weights)


def _evict(n, n_head_kv, hd, kv, block, keep, sink, recent):
    return dict(op="evict", n=n, n_head_kv=n_head_kv, hd=hd, kv=kv, block=block, keep=keep, sink=sink, recent=recent)


def listed():
    return [
        # one token of the 70B shape: only the launch counts
        dict(_rope("f32", 1, 64, 8, 128, 128, False, 32768, 1.0), name="rope 70b x1"),
        # a prompt chunk of the falcon shape in half precision, half of each head rotated, far behind the trained context
        dict(_rope("f16", 1901, 128, 8, 64, 32, True, 131072, 16.0), name="rope 40b yarn 1901"),
        # one token for each of 32 users with the 7B shape, in the middle of their blocks
        dict(_store("f16", 32, 1, 32, 128, 2048, 64), name="store 7b x32"),
        # a long prompt with the 70B shape
        dict(_store("f32", 1, 4096, 8, 128, 8192, 32), name="store 70b 4096"),
        # a chat's first tokens on a small draft model
        dict(_attention("f32", 1, 1, 4, 2, 64, 77, 16, False), name="attention small x1"),
        # one user with a long document, 70B shape
        dict(_attention("f32", 1, 1, 64, 8, 128, 32768, 64, False), name="attention 70b 32k x1"),
        # a full batch of users with the 7B shape (a KV head for each query head), each somewhere in a conversation
        dict(_attention("f16", 32, 1, 32, 32, 128, 2048, 64, False), name="attention 7b x32"),
        # a batch whose cache is kept at a budget: the weights are collected, 70B shape
        dict(_attention("f32", 8, 1, 64, 8, 128, 8000, 64, True), name="attention 70b weights x8"),
        # a chunk of a long prompt, 70B shape
        dict(_attention("f32", 1, 1024, 64, 8, 128, 4096, 32, False), name="attention 70b chunk 1024"),
        # the prompts of several users together, of different lengths, falcon shape in half precision
        dict(_attention("f16", 5, 701, 128, 8, 64, 1500, 64, False), name="attention 40b prompts x5"),
        # a long prompt is cut to what a small budget holds, 70B shape
        dict(_evict(1, 8, 128, 16384, 64, 2048, 4, 256), name="evict 70b 16k to 2k"),
        # a batch at its budget, 7B shape: the slots of the last 256 tokens are made free again
        dict(_evict(16, 32, 128, 1280, 32, 1024, 4, 256), name="evict 7b 1280 to 1024 x16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= 0.7 * most:
            return c


def _draw(rng):
    op = rng.choice(["rope", "store", "attention", "attention", "attention", "evict"])
    x, hd, block = rng.choice(["f32", "f16"]), rng.choice([64, 64, 96, 128, 128, 128, 192, 256]), rng.choice([16, 32, 64, 128])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 7, 8, 8, 16])
    if op == "rope":
        return _rope(x, _log(rng, 1, 4096), kv_heads * group, kv_heads, hd, hd if rng.random() < 0.6 else rng.randint(1, hd // 2) * 2, rng.random() < 0.5,
                     _log(rng, 100, 1000000), rng.choice([1.0, 1.0, 2.0, 8.0, 32.0]))
    if op == "store":
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        n = _log(rng, 1, 64) if new == 1 else _log(rng, 1, max(1, 8192 // new)) if new < 1024 else 1
        return _store(x, n, new, kv_heads, hd, -(-(new + rng.randint(0, 2000)) // 128) * 128, block)
    if op == "evict":
        keep = _log(rng, 1, 32) * 128
        return _evict(_log(rng, 1, 32), kv_heads, hd, keep + _log(rng, 1, 12000), block, keep, rng.randint(0, 16), rng.randint(0, keep // 2))
    kind = rng.choice(["decode", "decode", "few", "prompt"])
    if kind == "decode":
        return _attention(x, _log(rng, 1, 48), 1, kv_heads * group, kv_heads, hd, _log(rng, 1, 40000), block, rng.random() < 0.3)
    if kind == "few":
        new = rng.randint(2, 24)
        return _attention(x, _log(rng, 1, 12), new, kv_heads * group, kv_heads, hd, new + _log(rng, 1, 20000), block, rng.random() < 0.3)
    new = _log(rng, 25, 2048)
    return _attention(x, _log(rng, 1, 6), new, kv_heads * group, kv_heads, hd, new + rng.choice([0, _log(rng, 1, 6000)]), block, rng.random() < 0.2)


# ---------------------------------------------------------------------------------------------- sizes

def _cost(case):
    w = work(case)
    kv = 0
    if case["op"] in ("attention", "evict"):
        kv = 10.0 * case["n"] * case["n_head_kv"] * (case["kv"] + 128) * case["hd"]
        if case["op"] == "attention" and case["n"] * case["new"] * case["n_head"] * case["kv"] > 8e8:        # what a plain form has to hold
            return math.inf
    return w["bytes"] + w["flops"] / 100 + kv


def _n_ctx(case):
    return case["n_ctx"] if case["op"] == "store" else -(-case["kv"] // 128) * 128


def _news(case):
    """New tokens of each sequence: the first has the most."""
    return [case["new"] - i * (case["new"] - 1) // (2 * case["n"]) for i in range(case["n"])]


def _lens(case):
    """Slots of each sequence, its new tokens among them: the first has the most, the last about half of that."""
    if case["op"] == "evict":
        return [case["kv"] - i * (case["kv"] // 4) // case["n"] for i in range(case["n"])]
    if case["op"] == "store":
        return [case["n_ctx"] - (i * 29 + 11) % (case["n_ctx"] - new + 1) for i, new in enumerate(_news(case))]
    return [max(new, case["kv"] - i * (case["kv"] // 2) // case["n"]) for i, new in enumerate(_news(case))]


def work(case):
    if case["op"] == "rope":
        values = case["T"] * (case["n_head"] + case["n_head_kv"]) * case["hd"]
        return {"bytes": 2 * values * (4 if case["x"] == "f32" else 2) + 4 * case["T"], "flops": 3.0 * values * case["n_rot"] / case["hd"]}
    H, hd, B = case["n_head_kv"], case["hd"], case["block"]
    size = 4 if case.get("x") == "f32" else 2
    if case["op"] == "store":
        # the new rows once, codes of the touched blocks written, those of earlier tokens read, and all of them read back as values
        new, first = sum(_news(case)), [n - m for n, m in zip(_lens(case), _news(case))]
        old = sum(p % B for p in first)
        blocks = sum(-(-n // B) - p // B for n, p in zip(_lens(case), first))
        return {"bytes": 2 * H * (new * hd * size + (new + 2 * old) * hd + 12 * blocks + (new + old) * hd * 5), "flops": 4.0 * 2 * H * (new + old) * hd}
    if case["op"] == "evict":
        # weights of all slots; with weights that do not go by the slot, the share of the budget that comes from behind it moves
        bytes_ = 0
        for n in _lens(case):
            if n > case["keep"]:
                least = case["sink"] + case["recent"]
                share = (case["keep"] - least) / max(1, n - least)
                moved = case["recent"] + share * max(0, n - case["keep"] - case["recent"]) if case["recent"] <= n - case["keep"] else n - case["keep"]
                bytes_ += H * (4 * n + 2 * moved * 2 * hd)
            bytes_ += H * min(n, case["keep"]) * (8 + 2 * 5 * hd)                                            # weights and slots out, values read back
        return {"bytes": float(bytes_), "flops": float(bytes_) / 4}
    keys = sum(_lens(case))
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(_lens(case), _news(case)))
    bytes_ = 2 * H * keys * hd + 8 * H * keys // B + 2 * sum(_news(case)) * case["n_head"] * hd * size
    if case["weights"]:
        bytes_ += 8 * H * keys
    return {"bytes": float(bytes_), "flops": 4.0 * hd * case["n_head"] * pairs}


# ---------------------------------------------------------------------------------------------- preparation

def _freqs(n_rot, scale):
    """(angle per position of each pair, factor of the rotated values): YaRN where the context is stretched by `scale`."""
    f = [BASE ** (-2.0 * i / n_rot) for i in range(n_rot // 2)]
    if scale == 1.0:
        return f, 1.0

    def pair(turns):                                                  # the pair that makes so many turns in the original context
        return n_rot * math.log(ORIG_CTX / (turns * 2 * math.pi)) / (2 * math.log(BASE))

    low, high = max(0, math.floor(pair(32.0))), min(n_rot - 1, math.ceil(pair(1.0)))
    keep = [1.0 - min(1.0, max(0.0, (i - low) / max(0.001, high - low))) for i in range(n_rot // 2)]
    return [x * (k + (1.0 - k) / scale) for x, k in zip(f, keep)], 1.0 + 0.1 * math.log(scale)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(case)
    if case["op"] == "rope":
        dt = TYPES[case["x"]]
        # queries and keys as the projections leave them: rows of one matrix, the values behind them
        qkv = torch.randn(case["T"], (case["n_head"] + 2 * case["n_head_kv"]) * case["hd"], device="cuda", generator=gen).to(dt)
        nq, nk = case["n_head"] * case["hd"], case["n_head_kv"] * case["hd"]
        f, mscale = _freqs(case["n_rot"], case["scale"])
        start = case["far"] - case["T"]
        state.update(q=qkv[:, :nq], k=qkv[:, nq:nq + nk], freqs=torch.tensor(f, dtype=torch.float64, device="cuda"), mscale=mscale,
                     pos=torch.arange(max(0, start), max(0, start) + case["T"], dtype=torch.int32, device="cuda"))
        return state
    n, H, hd, n_ctx = case["n"], case["n_head_kv"], case["hd"], _n_ctx(case)
    # codes as a store leaves them: normal values over four standard deviations, scales of blocks within a factor of each other
    for name in ("k", "v"):
        state[name + "_codes"] = (torch.randn(n, H, n_ctx, hd, device="cuda", generator=gen) * 30.0).round_().clamp_(-127, 127).to(torch.int8)
        state[name + "_scale"] = torch.exp(torch.randn(n, H, n_ctx // case["block"], device="cuda", generator=gen) * 0.4) * (1.0 / 30.0)
    # sequences lie in the cache in another order than in the batch
    state["seq"] = torch.randperm(n, device="cuda", generator=gen).to(torch.int32)
    lens = _lens(case)
    if case["op"] == "evict":
        state["lens"] = _ints(lens)
        # accumulated weights: a few slots have most of them
        state["weights"] = torch.exp(torch.randn(n, H, n_ctx, device="cuda", generator=gen) * 2.0)
        state["weights_out"] = torch.zeros_like(state["weights"])
        state.update(all_start=_ints([i * case["keep"] for i in range(n + 1)]), all_pos=_ints([0] * n))
        return state
    news = _news(case)
    state["q_start"], state["pos0"] = _ints([sum(news[:i]) for i in range(n + 1)]), _ints([a - b for a, b in zip(lens, news)])
    dt, T = TYPES[case["x"]], sum(news)
    if case["op"] == "store":
        state["k"], state["v"] = (torch.randn(T, H * hd, device="cuda", generator=gen).to(dt) for _ in range(2))
        # the touched blocks from their first slots on, to be read back
        first = [(a - b) // case["block"] * case["block"] for a, b in zip(lens, news)]
        span = [a - f for a, f in zip(lens, first)]
        state.update(back_start=_ints([sum(span[:i]) for i in range(n + 1)]), back_pos=_ints(first), back_rows=sum(span), back_most=max(span))
        return state
    state["q"] = torch.randn(T, case["n_head"] * hd, device="cuda", generator=gen).to(dt)
    state["T"], state["max_kv"] = T, max(lens)
    if case["weights"]:
        state["weights_in"] = torch.rand(n, H, n_ctx, device="cuda", generator=gen)
        state["weights_out"] = torch.zeros(n, H, n_ctx, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------- the pass

def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "store": _plain_store, "attention": _plain_attention, "evict": _plain_evict}[state["op"]](state)


def _run_own(s):
    from powerinfer_b200 import ggml_ops as g
    if s["op"] == "rope":
        q, k = g.rope_ext(s["q"], s["k"], s["pos"], g.RopeFreqs(s["freqs"], s["mscale"]), s["hd"], mode=2 if s["halves"] else 0)
        return {"q": q, "k": k}
    cache = g.KvCacheQ8(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    if s["op"] == "store":
        g.kv_store_q8(cache, s["k"], s["v"], s["q_start"], s["pos0"], s["seq"], max_new=s["new"])
        k, v = g.kv_load_q8(cache, s["back_start"], s["back_pos"], s["back_rows"], s["seq"], max_new=s["back_most"])
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if s["op"] == "attention":
        out = g.attention_q8(cache, s["q"], s["q_start"], s["pos0"], s["seq"], max_new=s["new"], max_kv=s["max_kv"], weights_in=s.get("weights_in"),
                             weights_out=s.get("weights_out"))
        return {"out": out, "weights": s["weights_out"]} if s["weights"] else {"out": out}
    kept = g.kv_evict_q8(cache, s["weights"], s["lens"], s["keep"], n_sink=s["sink"], n_recent=s["recent"], seq=s["seq"], weights_out=s["weights_out"])
    k, v = g.kv_load_q8(cache, s["all_start"], s["all_pos"], s["n"] * s["keep"], s["seq"], max_new=s["keep"])
    return {"kept": kept, "weights": s["weights_out"], "k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_rope(s):
    half = s["n_rot"] // 2
    a = s["pos"].double()[:, None] * s["freqs"][None, :]
    c, sn = (torch.cos(a) * s["mscale"]).float()[:, None], (torch.sin(a) * s["mscale"]).float()[:, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].float().reshape(s["T"], -1, s["hd"])
        y = x.clone()
        if s["halves"]:
            x0, x1 = x[..., :half], x[..., half:2 * half]
            y[..., :half], y[..., half:2 * half] = x0 * c - x1 * sn, x0 * sn + x1 * c
        else:
            x0, x1 = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            y[..., 0:2 * half:2], y[..., 1:2 * half:2] = x0 * c - x1 * sn, x0 * sn + x1 * c
        out[name] = y.to(s[name].dtype).reshape(s["T"], -1)
    return out


def _codes(x, inv):
    """rne(x * inv) within 127; what is not a number is 0"""
    return torch.nan_to_num(x * inv, nan=0.0, posinf=127.0, neginf=-127.0).clamp_(-127, 127).round_()


def _inverse(s):
    return torch.where(s >= torch.finfo(torch.float32).tiny, 1.0 / s, torch.zeros_like(s))


def _rows_of(codes, scale, start, pos, seq, rows, block):
    """Values of the slots pos[i].. of sequence seq[i], as many as start says: [rows, heads, hd]"""
    at = torch.arange(rows, device="cuda", dtype=torch.int32)
    i = torch.searchsorted(start[1:].contiguous(), at, right=True)
    slot = (pos[i] + at - start[i]).long()
    which = seq[i].long()
    return codes[which, :, slot].float() * scale[which, :, slot // block][..., None]


def _plain_store(s):
    B, H, hd = s["block"], s["n_head_kv"], s["hd"]
    seq, n_new = s["seq"].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    first, pos = s["q_start"][:-1].long(), s["pos0"].long()
    nb = (s["new"] + 2 * B - 2) // B                                   # blocks that so many tokens can touch
    block = pos[:, None] // B + torch.arange(nb, device="cuda")
    slot = block[..., None] * B + torch.arange(B, device="cuda")       # [n, nb, B]
    new = (slot >= pos[:, None, None]) & (slot < (pos + n_new)[:, None, None])
    old = (slot < pos[:, None, None]) & new.any(-1, keepdim=True)
    token = torch.where(new, first[:, None, None] + slot - pos[:, None, None], 0)
    inside = block.clamp(max=s["n_ctx"] // B - 1)
    for name in ("k", "v"):
        codes, scale = s[name + "_codes"].view(-1, H, s["n_ctx"] // B, B, hd), s[name + "_scale"]
        x = s[name].float().view(-1, H, hd)[token]                     # [n, nb, B, H, hd]
        size = torch.where(new[..., None, None] & torch.isfinite(x), x.abs(), 0).amax((2, 4))
        before = torch.where(old.any(-1)[..., None], scale[seq[:, None], :, inside], torch.zeros_like(size))
        now = torch.maximum(size / 127.0, before)
        kept = codes[seq[:, None], :, inside].transpose(2, 3)          # [n, nb, B, H, hd]
        ratio = torch.where(now > 0, before / now, torch.ones_like(now))
        moved = (kept.float() * ratio[:, :, None, :, None]).round_()
        fresh = _codes(x, _inverse(now)[:, :, None, :, None])
        got = torch.where(new[..., None, None], fresh, torch.where(old[..., None, None], moved, kept.float())).to(torch.int8).transpose(2, 3)
        touched = new.any(-1)
        a, b = (seq[:, None] + torch.zeros_like(block))[touched], block[touched]
        codes[a, :, b] = got[touched]
        scale[a, :, b] = now[touched]
    out = {name: _rows_of(s[name + "_codes"], s[name + "_scale"], s["back_start"], s["back_pos"], s["seq"], s["back_rows"], B) for name in ("k", "v")}
    return {"k": out["k"].reshape(-1, H * hd), "v": out["v"].reshape(-1, H * hd), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(s):
    n, new, H, hd, kv = s["n"], s["new"], s["n_head_kv"], s["hd"], s["max_kv"]
    seq, group = s["seq"].long(), s["n_head"] // H
    j = torch.arange(new, device="cuda")
    n_new = (s["q_start"][1:] - s["q_start"][:-1])[:, None]
    real = j < n_new                                                   # [n, new]: the padded batch's own rows
    row = torch.where(real, s["q_start"][:-1, None] + j, 0).long()
    q = s["q"].float().view(-1, H, group, hd)[row].permute(0, 2, 3, 1, 4).reshape(n, H, group * new, hd)

    def values(name):
        scale = s[name + "_scale"].repeat_interleave(s["block"], 2)[seq, :, :kv, None]
        return s[name + "_codes"][seq, :, :kv].float() * scale

    score = (q @ values("k").transpose(2, 3)) * (1.0 / math.sqrt(hd))
    seen = torch.arange(kv, device="cuda") <= (s["pos0"][:, None] + j)[..., None]                             # [n, new, kv]
    score = score.view(n, H, group, new, kv).masked_fill_(~(seen & real[..., None])[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    p = p / p.sum(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).tiny)
    o = (p.view(n, H, group * new, kv) @ values("v")).view(n, H, group, new, hd).permute(0, 3, 1, 2, 4)
    out = torch.empty(s["T"], H, group, hd, device="cuda")
    out[row[real]] = o[real]
    out = {"out": out.view(s["T"], -1).to(s["q"].dtype)}
    if s["weights"]:
        slot = torch.arange(kv, device="cuda")
        had = torch.where((slot < s["pos0"][:, None])[:, None], s["weights_in"][seq, :, :kv], 0.0)
        end = (slot < s["pos0"][:, None] + n_new)[:, None]
        s["weights_out"][seq, :, :kv] = torch.where(end, had + p.sum((2, 3)), s["weights_out"][seq, :, :kv])
        out["weights"] = s["weights_out"]
    return out


def _plain_evict(s):
    n, H, hd, B, keep = s["n"], s["n_head_kv"], s["hd"], s["block"], s["keep"]
    seq, lens = s["seq"].long(), s["lens"][:, None, None]
    n_ctx = s["weights"].shape[2]
    w = s["weights"][seq]
    slot = torch.arange(n_ctx, device="cuda")
    inside = slot < lens
    sure = inside & ((slot < s["sink"]) | (slot >= lens - s["recent"]))
    key = torch.where(sure, math.inf, torch.where(inside, w, -1.0))
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    chosen = torch.zeros_like(key, dtype=torch.bool).scatter_(2, order[..., :keep], True) & inside             # lowest slots first among equals
    low, high = chosen[..., :keep], chosen[..., keep:]
    hole = ~low & inside[..., :keep]
    # the r-th hole takes the r-th kept slot behind the budget
    rank = hole.cumsum(-1)
    place = torch.where(high, high.cumsum(-1), 0)
    from_rank = torch.zeros(n, H, n_ctx + 1, dtype=torch.int64, device="cuda").scatter_(2, place, slot[keep:].expand_as(place))
    kept = torch.where(hole, torch.gather(from_rank, 2, rank), slot[:keep].expand_as(hole))
    kept = torch.where(inside[..., :keep].expand_as(kept), kept, -1)
    source, live = kept.clamp(min=0), (kept >= 0)
    s["weights_out"][seq, :, :keep] = torch.where(live, torch.gather(w, 2, source), s["weights_out"][seq, :, :keep])
    moves = (hole.view(n, H, keep // B, B)).any(-1)                     # blocks that take a row from elsewhere
    for name in ("k", "v"):
        codes, scale = s[name + "_codes"][seq], s[name + "_scale"][seq]
        rows = torch.gather(codes[..., :, :], 2, source[..., None].expand(n, H, keep, hd)).float()
        of_row = torch.where(live, torch.gather(scale, 2, source // B), 0.0)
        now = torch.where(moves, of_row.view(n, H, keep // B, B).amax(-1), scale[..., :keep // B])
        ratio = torch.where(live, of_row / now.repeat_interleave(B, 2), 1.0)
        got = torch.where((moves.repeat_interleave(B, 2) & live)[..., None], (rows * ratio[..., None]).round_(), codes[..., :keep, :].float()).to(torch.int8)
        s[name + "_codes"][seq, :, :keep] = got
        s[name + "_scale"][seq, :, :keep // B] = now
    out = {name: _rows_of(s[name + "_codes"], s[name + "_scale"], s["all_start"], s["all_pos"], s["seq"], n * keep, B).reshape(-1, H * hd) for name in ("k", "v")}
    return {"kept": kept.to(torch.int32), "weights": s["weights_out"], **out, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# ---------------------------------------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "store": _exact_store, "attention": _exact_attention, "evict": _exact_evict}[case["op"]](s)


def _exact_rope(s):
    """Each pair as a complex number, turned."""
    half = s["n_rot"] // 2
    turn = torch.polar(torch.full((s["T"], half), s["mscale"], dtype=torch.float64, device="cuda"), torch.outer(s["pos"].double(), s["freqs"]))
    out = {}
    for name in ("q", "k"):
        x = s[name].double().reshape(s["T"], -1, s["hd"])
        head, rest = x[..., :2 * half], x[..., 2 * half:]
        pairs = head.unflatten(-1, (2, half)).transpose(-1, -2) if s["halves"] else head.unflatten(-1, (half, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
        head = z.transpose(-1, -2).flatten(-2) if s["halves"] else z.flatten(-2)
        out[name] = torch.cat([head, rest], -1).reshape(s["T"], -1)
    return out


def _host(s, *names):
    return [s[n].cpu().numpy() for n in names]


def _exact_store(s):
    """Block by block.  Codes and scales are defined by their steps in 32 bits; the values that they stand for are in 64."""
    q_start, pos0, seq = _host(s, "q_start", "pos0", "seq")
    B, H, hd, one = s["block"], s["n_head_kv"], s["hd"], np.float32(1.0)
    out = {}
    for name in ("k", "v"):
        x, codes, scale = _host(s, name, name + "_codes", name + "_scale")
        x, back = x.astype(np.float32).reshape(-1, H, hd), []
        for i in range(s["n"]):
            p, m = int(pos0[i]), int(q_start[i + 1] - q_start[i])
            for b in range(p // B, (p + m - 1) // B + 1):
                lo, hi = max(p, b * B), min(p + m, (b + 1) * B)
                new = x[q_start[i] + lo - p:q_start[i] + hi - p].transpose(1, 0, 2)                          # [H, rows, hd]
                had = codes[seq[i], :, b * B:lo]
                was = scale[seq[i], :, b].copy() if lo > b * B else np.zeros(H, np.float32)
                now = np.maximum(np.abs(new).max((1, 2)) / np.float32(127.0), was)
                if lo > b * B:
                    codes[seq[i], :, b * B:lo] = np.rint(had.astype(np.float32) * (was / now)[:, None, None])
                codes[seq[i], :, lo:hi] = np.clip(np.rint(new * (one / now)[:, None, None]), -127, 127)
                scale[seq[i], :, b] = now
                back.append((codes[seq[i], :, b * B:hi].astype(np.float64) * now.astype(np.float64)[:, None, None]).transpose(1, 0, 2).reshape(-1, H * hd))
        out[name], out[name + "_scale"] = np.concatenate(back), scale.astype(np.float64)
    return out


def _exact_attention(s):
    """Sequence by sequence, KV head by KV head."""
    q_start, pos0, seq = _host(s, "q_start", "pos0", "seq")
    H, hd, group = s["n_head_kv"], s["hd"], s["n_head"] // s["n_head_kv"]
    if work(s)["flops"] > 4e12:                                        # over a few seconds in 64 bits
        return None
    out = torch.zeros(s["T"], H, group, hd, dtype=torch.float64, device="cuda")
    weights = s["weights_out"].double() if s["weights"] else None
    for i in range(s["n"]):
        p, a, b = int(pos0[i]), int(q_start[i]), int(q_start[i + 1])
        n = p + b - a
        late = torch.arange(n, device="cuda")[None] > p + torch.arange(b - a, device="cuda")[:, None]
        for h in range(H):
            k, v = (s[x + "_codes"][seq[i], h, :n].double() * s[x + "_scale"][seq[i], h].double().repeat_interleave(s["block"])[:n, None] for x in ("k", "v"))
            score = torch.einsum("tgd,jd->gtj", s["q"][a:b].double().view(b - a, H, group, hd)[:, h], k) / math.sqrt(hd)
            p_ = torch.softmax(score.masked_fill(late, -math.inf), -1)
            out[a:b, h] = torch.einsum("gtj,jd->tgd", p_, v)
            if weights is not None:
                weights[seq[i], h, :n] = p_.sum((0, 1))
                weights[seq[i], h, :p] += s["weights_in"][seq[i], h, :p].double()
    out = {"out": out.view(s["T"], -1)}
    return out if weights is None else {**out, "weights": weights}


def _exact_evict(s):
    """Sequence by sequence, KV head by KV head; codes and scales by their steps in 32 bits, as the store's."""
    lens, seq, w = _host(s, "lens", "seq", "weights")
    B, H, hd, keep = s["block"], s["n_head_kv"], s["hd"], s["keep"]
    w_out = s["weights_out"].cpu().numpy().astype(np.float64)
    kept = np.full((s["n"], H, keep), -1, np.int32)
    for i, n in enumerate(lens):
        for h in range(H):
            kept[i, h, :min(n, keep)] = np.arange(min(n, keep))
            if n > keep:
                rank = w[seq[i], h, :n].astype(np.float64)
                rank[:s["sink"]] = np.inf
                rank[max(0, n - s["recent"]):] = np.inf
                best = np.zeros(n, bool)
                best[np.lexsort((np.arange(n), -rank))[:keep]] = True
                kept[i, h, np.flatnonzero(~best[:keep])] = keep + np.flatnonzero(best[keep:])
            m = min(n, keep)
            w_out[seq[i], h, :m] = w[seq[i], h, kept[i, h, :m]]
    out = {"kept": kept, "weights": w_out}
    for name in ("k", "v"):
        codes, scale = _host(s, name + "_codes", name + "_scale")
        new, new_scale = codes[:, :, :keep].copy(), scale.copy()
        for i in range(s["n"]):
            for h in range(H):
                for b in np.unique(np.flatnonzero(kept[i, h] > np.arange(keep)) // B):
                    rows = kept[i, h, b * B:(b + 1) * B]
                    of = scale[seq[i], h, rows // B]
                    new_scale[seq[i], h, b] = of.max()
                    new[seq[i], h, b * B:(b + 1) * B] = np.rint(codes[seq[i], h, rows].astype(np.float32) * (of / of.max())[:, None])
        stands = new[seq].astype(np.float64) * np.repeat(new_scale[seq][:, :, :keep // B], B, 2)[..., None].astype(np.float64)
        out[name], out[name + "_scale"] = stands.transpose(0, 2, 1, 3).reshape(-1, H * hd), new_scale.astype(np.float64)
    return out
