"""What is timed when the operators of drafted tokens over a paged cache are timed: one step of speculative decoding is a tree of drafted
tokens for each sequence, whose keys and values go into the cache, whose queries see the context and their own ancestors, and of which
the accepted path stays.

Four kinds of case, by `op`:

    append      keys and values of up to `new` tokens for each of n sequences into the pages of a cache, keys and queries rotated to their
                positions on the way (`halves`: pairs (i, i + n_rot/2), else (2i, 2i + 1)); `tree`: a token's position goes by its depth
    attention   up to `new` queries for each of n sequences of up to `kv` slots; `tree`: a token sees the context and its ancestors among
                the new ones, else it sees all before it
    tree        the parents of up to `new` drafted tokens for each of n sequences made into masks and positions, and, when the target
                model has made its choice behind each of them, the path that agrees with it
    keep        the path's `depth` rows moved up behind the context, in all layers of the cache

A cache is two pools, float16 [n_layer, n_pages, n_head_kv, page, hd], and a table, int32 [n, max_pages]: slot j of a sequence is row j % page of the
page that its table names at j // page.  The new tokens of sequence i are rows q_start[i] .. q_start[i+1] of q / k / v, in slots
pos0[i] and on; a token's parent is the number of an earlier one of its sequence, -1 for the root.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16}
BASE = 10000.0


def _append(x, n, new, n_head, n_head_kv, hd, kv, page, tree, n_rot, halves):
    return dict(op="append", x=x, n=n, new=new, n_head=n_head, n_head_kv=n_head_kv, hd=hd, kv=kv, page=page, tree=tree, n_rot=n_rot, halves=halves)


def _attention(x, n, new, n_head, n_head_kv, hd, kv, page, tree):
    return dict(op="attention", x=x, n=n, new=new, n_head=n_head, n_head_kv=n_head_kv, hd=hd, kv=kv, page=page, tree=tree)


def _tree(n, new):
    return dict(op="tree", n=n, new=new)


def _keep(n, new, depth, n_layer, n_head_kv, hd, kv, page):
    return dict(op="keep", n=n, new=new, depth=depth, n_layer=n_layer, n_head_kv=n_head_kv, hd=hd, kv=kv, page=page)


def listed():
    return [
        # the drafted trees of a few users, 70B shape: only the launch counts
        dict(_append("f32", 8, 25, 64, 8, 128, 500, 64, True, 128, False), name="append 70b trees x8"),
        # chunks of several prompts, falcon shape in half precision
        dict(_append("f16", 4, 1024, 128, 8, 64, 2000, 16, False, 64, True), name="append 40b prompts x4"),
        # a chat's first tokens on a small draft model
        dict(_attention("f32", 1, 1, 4, 2, 64, 77, 16, False), name="attention small x1"),
        # a full batch of users with the 7B shape (a KV head for each query head), each somewhere in a conversation, nothing drafted
        dict(_attention("f16", 32, 1, 32, 32, 128, 2048, 64, False), name="attention 7b x32"),
        # one user with a long document and a drafted tree, 70B shape
        dict(_attention("f32", 1, 25, 64, 8, 128, 32768, 64, True), name="attention 70b 32k tree"),
        # some users' trees with the 7B shape
        dict(_attention("f16", 8, 48, 32, 32, 128, 2000, 16, True), name="attention 7b trees x8"),
        # many users' trees, falcon shape in half precision
        dict(_attention("f16", 16, 32, 128, 8, 64, 1500, 64, True), name="attention 40b trees x16"),
        # a chunk of a long prompt into the paged cache, 70B shape
        dict(_attention("f32", 1, 1024, 64, 8, 128, 4096, 32, False), name="attention 70b chunk 1024"),
        # one user's tree
        dict(_tree(1, 25), name="tree x1"),
        # a full batch of large trees
        dict(_tree(64, 192), name="tree 192 x64"),
        # one user's accepted tokens, 7B shape
        dict(_keep(1, 25, 4, 32, 32, 128, 500, 64), name="keep 7b x1"),
        # a batch's accepted tokens, 70B shape
        dict(_keep(8, 32, 6, 80, 8, 128, 250, 64), name="keep 70b x8"),
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
    op = rng.choice(["append", "attention", "attention", "attention", "tree", "keep"])
    x, hd, page = rng.choice(["f32", "f16"]), rng.choice([64, 64, 96, 128, 128, 128, 192, 256]), rng.choice([16, 32, 64, 128])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8, 8, 16, 32]), rng.choice([1, 1, 2, 3, 4, 7, 8, 8, 16])
    if op == "tree":
        return _tree(_log(rng, 1, 64), _log(rng, 1, 256))
    if op == "keep":
        new = _log(rng, 2, 128)
        return _keep(_log(rng, 1, 32), new, rng.randint(1, min(new - 1, 12)), _log(rng, 1, 80), kv_heads, hd, new + _log(rng, 1, 1000), page)
    kind = rng.choice(["decode", "tree", "tree", "prompt"])
    new = 1 if kind == "decode" else _log(rng, 2, 192) if kind == "tree" else _log(rng, 25, 2048)
    n = _log(rng, 1, 48) if kind == "decode" else _log(rng, 1, 16) if kind == "tree" else _log(rng, 1, 6)
    if op == "append":
        return _append(x, n, new, kv_heads * group, kv_heads, hd, new + _log(rng, 1, 2000), page, kind == "tree", hd if rng.random() < 0.6 else rng.randint(1, hd // 2) * 2,
                       rng.random() < 0.5)
    kv = new + (_log(rng, 1, 30000) if new == 1 else rng.choice([0, _log(rng, 1, 6000)]) if kind == "prompt" else _log(rng, 1, 12000))
    return _attention(x, n, new, kv_heads * group, kv_heads, hd, kv, page, kind == "tree")


# ---------------------------------------------------------------------------------------------- sizes

def _cost(case):
    w = work(case)
    pools = 0 if case["op"] == "tree" else 8.0 * case.get("n_layer", 1) * case["n"] * case["n_head_kv"] * (case["kv"] + 128) * case["hd"]
    if case["op"] == "attention" and case["n"] * case["new"] * case["n_head"] * case["kv"] > 8e8:                 # what a plain form has to hold
        return math.inf
    if pools > 4e9:
        return math.inf
    return w["bytes"] + w["flops"] / 100 + pools


def _news(case):
    """New tokens of each sequence: the first has the most."""
    return [case["new"] - i * (case["new"] - 1) // (2 * case["n"]) for i in range(case["n"])]


def _lens(case):
    """Slots of each sequence, its new tokens among them: the first has the most, the last about half of that."""
    return [max(new, case["kv"] - i * (case["kv"] // 2) // case["n"]) for i, new in enumerate(_news(case))]


def work(case):
    news = _news(case)
    T = sum(news)
    if case["op"] == "tree":
        # parents, tokens and choices; masks and positions, paths (their ends alone, as they are a few tokens)
        return {"bytes": 4.0 * 3 * T + T * (8.0 * _words(case) + 4) + 8.0 * case["n"], "flops": 2.0 * T * (1 + math.log(case["new"]))}
    H, hd = case["n_head_kv"], case["hd"]
    if case["op"] == "keep":
        bytes_ = 4.0 * case["n"] * (case["depth"] + 1) + case["n"] * case["depth"] * case["n_layer"] * H * 2 * 2 * hd * 2.0
        return {"bytes": bytes_, "flops": bytes_ / 4}
    size = 4 if case["x"] == "f32" else 2
    if case["op"] == "append":
        values = T * (case["n_head"] + H) * hd
        return {"bytes": T * (2.0 * case["n_head"] * hd * size + 2 * H * hd * (size + 2) + 4), "flops": 3.0 * values * case["n_rot"] / hd}
    lens = _lens(case)
    if case["tree"]:                                                  # a token of a tree has 1 + ln of its number ancestors, itself among them
        pairs = sum(m * (n - m) + m * (1 + math.log(m)) for n, m in zip(lens, news))
    else:
        pairs = sum(m * (n - m) + m * (m + 1) / 2 for n, m in zip(lens, news))
    return {"bytes": 2.0 * H * sum(lens) * hd * 2 + 2.0 * T * case["n_head"] * hd * size + (8.0 * T * _words(case) if case["tree"] else 0), "flops": 4.0 * hd * case["n_head"] * pairs}


def _words(case):
    return -(-case["new"] // 64)


# ---------------------------------------------------------------------------------------------- preparation

def _ints(v):
    return torch.as_tensor(np.asarray(v, np.int32), device="cuda")


def _parents(news, seed):
    """Each token's parent is one of those before it in its sequence, any of them alike: most are near the root, some paths are long."""
    rng = random.Random(seed)
    return [[-1] + [rng.randrange(u) for u in range(1, m)] for m in news]


def _ancestors(parents):
    """[i][t, u]: whether token u of sequence i is t or one of its ancestors"""
    out = []
    for of in parents:
        a = np.eye(len(of), dtype=bool)
        for t, u in enumerate(of):
            if u >= 0:
                a[t] |= a[u]
        out.append(a)
    return out


def _mask_words(ancestors, words):
    rows = []
    for a in ancestors:
        bits = np.zeros((len(a), words * 64), np.uint8)
        bits[:, :len(a)] = a
        rows.append(np.packbits(bits, axis=1, bitorder="little").view(np.int64))
    return torch.as_tensor(np.concatenate(rows), device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state, n, news = dict(case), case["n"], _news(case)
    T = sum(news)
    state["q_start"], state["T"] = _ints(np.concatenate([[0], np.cumsum(news)])), T
    parents = _parents(news, seed)
    state["parents"] = _ints(sum(parents, []))
    if case["op"] == "tree":
        rng = random.Random(seed + 1)
        state["pos0"] = _ints([rng.randint(1, 4000) for _ in news])
        # drafted tokens, siblings different from each other for the most part; the target model chooses one of the drafted ones two times in three
        tokens = [[rng.randrange(32000) for _ in range(m)] for m in news]
        choice = [[rng.randrange(32000) for _ in range(m)] for m in news]
        for of, tok, ch in zip(parents, tokens, choice):
            for u in range(len(of) - 1, 0, -1):
                if rng.random() < 0.66:
                    ch[of[u]] = tok[u]
        state["tokens"], state["choice"] = _ints(sum(tokens, [])), _ints(sum(choice, []))
        return state
    H, hd, page, lens = case["n_head_kv"], case["hd"], case["page"], _lens(case)
    pages = [-(-m // page) for m in lens]
    n_pages = sum(pages) + 3
    # a pool whose pages were used before, handed out in no order
    for name in ("k_pool", "v_pool"):
        state[name] = torch.randn(case.get("n_layer", 1), n_pages, H, page, hd, device="cuda", generator=gen, dtype=torch.float16)
    free = np.random.default_rng(seed).permutation(n_pages)
    table = np.full((n, max(pages)), -1, np.int32)
    for i, m in enumerate(pages):
        table[i, :m], free = free[:m], free[m:]
    state["table"] = _ints(table)
    # sequences lie in the table in another order than in the batch
    order = torch.randperm(n, device="cuda", generator=gen)
    state["seq"] = order.to(torch.int32)
    state["table"][order] = state["table"].clone()
    state["pos0"] = _ints([a - b for a, b in zip(lens, news)])
    if case["op"] == "keep":
        rng = random.Random(seed)
        paths = [[0] + sorted(rng.sample(range(1, m), min(m - 1, case["depth"]))) for m in news]
        state["n_path"] = _ints([len(p) for p in paths])
        state["path"] = _ints([p + [-1] * (case["new"] - len(p)) for p in paths])
        return state
    dt = TYPES[case["x"]]
    if case["op"] == "append":
        # queries, keys and values as the projections leave them: rows of one matrix
        qkv = torch.randn(T, (case["n_head"] + 2 * H) * hd, device="cuda", generator=gen).to(dt)
        nq, nk = case["n_head"] * hd, H * hd
        state.update(q=qkv[:, :nq], k=qkv[:, nq:nq + nk], v=qkv[:, nq + nk:])
        state["freqs"] = torch.tensor([BASE ** (-2.0 * i / case["n_rot"]) for i in range(case["n_rot"] // 2)], dtype=torch.float64, device="cuda")
        depth = [a.sum(1) - 1 if case["tree"] else np.arange(len(a)) for a in _ancestors(parents)]
        state["pos"] = _ints(np.concatenate([a - b + d for a, b, d in zip(lens, news, depth)]))
        return state
    state["q"] = torch.randn(T, case["n_head"] * hd, device="cuda", generator=gen).to(dt)
    state["max_kv"] = max(lens)
    state["mask"] = _mask_words(_ancestors(parents), _words(case)) if case["tree"] else None
    return state


# ---------------------------------------------------------------------------------------------- the pass

def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attention": _plain_attention, "tree": _plain_tree, "keep": _plain_keep}[state["op"]](state)


def _run_own(s):
    from powerinfer_b200 import ggml_ops as g
    if s["op"] == "tree":
        mask, pos = g.tree_mask(s["parents"], s["q_start"], s["pos0"], max_new=s["new"])
        path, n_path, then = g.tree_accept(s["tokens"], s["parents"], s["choice"], s["q_start"], max_new=s["new"])
        return {"mask": mask, "pos": pos, "path": path, "n_path": n_path, "next": then}
    cache = g.KvCachePaged(s["k_pool"], s["v_pool"], s["table"])
    if s["op"] == "append":
        q = g.kv_append_paged(cache, s["k"], s["v"], s["q_start"], s["pos0"], s["seq"], max_new=s["new"], q=s["q"], pos=s["pos"], freqs=g.RopeFreqs(s["freqs"]),
                              mode=2 if s["halves"] else 0)
        return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    if s["op"] == "attention":
        return {"out": g.attention_tree(cache, s["q"], s["q_start"], s["pos0"], s["seq"], max_new=s["new"], max_kv=s["max_kv"], mask=s["mask"])}
    g.kv_keep_paged(cache, s["path"], s["n_path"], s["pos0"], s["seq"])
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _token_of(s):
    """Of each row: the entry that it belongs to, and its number in it."""
    at = torch.arange(s["T"], device="cuda", dtype=torch.int32)
    i = torch.searchsorted(s["q_start"][1:].contiguous(), at, right=True)
    return i, at - s["q_start"][i]


def _place(s, i, slot):
    """Page and row of the slots of entries i."""
    slot = slot.long()
    return s["table"][s["seq"].long()[i], slot // s["page"]].long(), slot % s["page"]


def _plain_append(s):
    H, hd, half = s["n_head_kv"], s["hd"], s["n_rot"] // 2
    a = s["pos"].double()[:, None] * s["freqs"][None, :]
    c, sn = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]

    def turned(x):
        x = x.float().reshape(s["T"], -1, hd)
        y = x.clone()
        first, second = (slice(0, half), slice(half, 2 * half)) if s["halves"] else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
        x0, x1 = x[..., first], x[..., second]
        y[..., first], y[..., second] = x0 * c - x1 * sn, x0 * sn + x1 * c
        return y

    i, t = _token_of(s)
    page, row = _place(s, i, s["pos0"][i] + t)
    s["k_pool"][0][page, :, row] = turned(s["k"]).half()
    s["v_pool"][0][page, :, row] = s["v"].float().reshape(s["T"], H, hd).half()
    return {"q": turned(s["q"]).to(s["q"].dtype).reshape(s["T"], -1), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_attention(s):
    n, new, H, hd, kv = s["n"], s["new"], s["n_head_kv"], s["hd"], s["max_kv"]
    group = s["n_head"] // H
    i, t = _token_of(s)
    q = torch.zeros(n, new, H, group, hd, device="cuda")
    q[i, t.long()] = s["q"].float().view(-1, H, group, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, H, group * new, hd)
    slot = torch.arange(kv, device="cuda")
    inside = slot < (s["pos0"] + s["q_start"][1:] - s["q_start"][:-1])[:, None]
    page, row = _place(s, torch.arange(n, device="cuda")[:, None], slot[None, :])
    page = torch.where(inside, page, 0)

    def values(name):
        return torch.where(inside[..., None, None], s[name][0][page, :, row].float(), 0.0).transpose(1, 2)               # [n, H, kv, hd]

    score = (q @ values("k_pool").transpose(2, 3)) * (1.0 / math.sqrt(hd))
    u = slot[None, :] - s["pos0"][:, None]                                                                              # number among the new tokens
    seen = torch.zeros(n, new, kv, dtype=torch.bool, device="cuda")
    ui = u[i]
    if s["mask"] is None:
        seen[i, t.long()] = ui <= t[:, None]
    else:
        bit = ui.clamp(min=0, max=s["new"] - 1)
        seen[i, t.long()] = (ui < 0) | ((torch.gather(s["mask"], 1, bit // 64) >> (bit % 64)) & 1).bool() & (ui < s["new"])
    seen &= inside[:, None]
    score = score.view(n, H, group, new, kv).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    p = p / p.sum(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).tiny)
    o = (p.view(n, H, group * new, kv) @ values("v_pool")).view(n, H, group, new, hd).permute(0, 3, 1, 2, 4)
    return {"out": o[i, t.long()].reshape(s["T"], -1).to(s["q"].dtype)}


def _plain_tree(s):
    n, new = s["n"], s["new"]
    i, t = _token_of(s)
    t = t.long()

    def padded(v, fill):
        return torch.full((n, new), fill, dtype=torch.int64, device="cuda").index_put_((i, t), v.long())

    real = padded(torch.ones_like(s["parents"]), 0).bool()
    parent, number = padded(s["parents"], -1), torch.arange(new, device="cuda")
    link = (parent[..., None] == number).float()                      # [n, t, u]: u is t's parent
    reach = link + torch.eye(new, device="cuda")
    span = 1
    while span < new:                                                 # paths of twice the length
        reach, span = (reach @ reach).clamp_(max=1.0), span * 2
    sees = reach > 0
    words = -(-new // 64)
    bits = torch.zeros(n, new, words * 64, dtype=torch.int64, device="cuda")
    bits[..., :new] = sees
    mask = (bits.view(n, new, words, 64) << torch.arange(64, device="cuda")).sum(-1)
    pos = s["pos0"][:, None] + sees.sum(-1) - 1
    # a token is taken where it is what the target chose behind its parent, no earlier sibling was, and so are all of its ancestors; the root is
    agrees = (parent >= 0) & real & (padded(s["tokens"], -1) == torch.gather(padded(s["choice"], -2), 1, parent.clamp(min=0)))
    earlier = (parent[:, :, None] == parent[:, None, :]) & agrees[:, None, :] & (number[None, :] < number[:, None])
    good = agrees & ~earlier.any(-1)
    good[:, 0] = real[:, 0]
    taken = real & (~sees | good[:, None, :]).all(-1)
    order = torch.sort(torch.where(taken, number, new), dim=1)[0]
    n_path = taken.sum(1)
    last = torch.gather(order, 1, (n_path - 1).clamp(min=0)[:, None])
    then = torch.gather(padded(s["choice"], -1), 1, last.clamp(max=new - 1))[:, 0]
    return {"mask": mask[i, t], "pos": pos[i, t].int(), "path": torch.where(order < new, order, -1).int(), "n_path": n_path.int(), "next": then.int()}


def _plain_keep(s):
    r = torch.arange(s["path"].shape[1], device="cuda")
    i, r = torch.nonzero(r < s["n_path"][:, None], as_tuple=True)
    from_page, from_row = _place(s, i, s["pos0"][i] + s["path"][i, r])
    to_page, to_row = _place(s, i, s["pos0"][i] + r)
    for name in ("k_pool", "v_pool"):
        s[name][:, to_page, :, to_row] = s[name][:, from_page, :, from_row]
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"]}


# ---------------------------------------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "tree": _exact_tree, "keep": _exact_keep}[case["op"]](s)


def _host(s, *names):
    return [s[n].cpu().numpy() for n in names]


def _slots(s, i, lo, hi, host):
    """(pages, rows) of the slots lo .. hi - 1 of entry i; host: table and order of the sequences"""
    table, seq = host
    j = np.arange(lo, hi)
    return torch.as_tensor(table[seq[i], j // s["page"]].astype(np.int64), device="cuda"), torch.as_tensor(j % s["page"], device="cuda")


def _exact_append(s):
    """Each pair as a complex number, turned."""
    half, hd, H = s["n_rot"] // 2, s["hd"], s["n_head_kv"]
    turn = torch.polar(torch.ones(s["T"], half, dtype=torch.float64, device="cuda"), torch.outer(s["pos"].double(), s["freqs"]))

    def turned(x):
        x = x.double().reshape(s["T"], -1, hd)
        head, rest = x[..., :2 * half], x[..., 2 * half:]
        pairs = head.unflatten(-1, (2, half)).transpose(-1, -2) if s["halves"] else head.unflatten(-1, (half, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
        return torch.cat([z.transpose(-1, -2).flatten(-2) if s["halves"] else z.flatten(-2), rest], -1)

    k, v = turned(s["k"]), s["v"].double().reshape(s["T"], H, hd)
    q_start, pos0, *host = _host(s, "q_start", "pos0", "table", "seq")
    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    for i in range(s["n"]):
        a, b = int(q_start[i]), int(q_start[i + 1])
        page, row = _slots(s, i, int(pos0[i]), int(pos0[i]) + b - a, host)
        k_pool[0, page, :, row], v_pool[0, page, :, row] = k[a:b], v[a:b]
    return {"q": turned(s["q"]).reshape(s["T"], -1), "k_pool": k_pool, "v_pool": v_pool}


def _walk(parents, t):
    """t and its ancestors, from the root on"""
    way = []
    while t >= 0:
        way.append(t)
        t = int(parents[t])
    return way[::-1]


def _exact_attention(s):
    """Sequence by sequence, KV head by KV head."""
    if work(s)["flops"] > 4e12:                                       # over a few seconds in 64 bits
        return None
    q_start, pos0, parents, *host = _host(s, "q_start", "pos0", "parents", "table", "seq")
    H, hd, group = s["n_head_kv"], s["hd"], s["n_head"] // s["n_head_kv"]
    out = torch.zeros(s["T"], H, group, hd, dtype=torch.float64, device="cuda")
    for i in range(s["n"]):
        p, a, b = int(pos0[i]), int(q_start[i]), int(q_start[i + 1])
        m = b - a
        sees = np.zeros((m, p + m), bool)
        sees[:, :p] = True
        for t in range(m):
            sees[t, [p + u for u in (_walk(parents[a:b], t) if s["tree"] else range(t + 1))]] = True
        hidden = torch.as_tensor(~sees, device="cuda")
        page, row = _slots(s, i, 0, p + m, host)
        for h in range(H):
            k, v = (s[x][0, page, h, row].double() for x in ("k_pool", "v_pool"))
            score = torch.einsum("tgd,jd->gtj", s["q"][a:b].double().view(m, H, group, hd)[:, h], k) / math.sqrt(hd)
            out[a:b, h] = torch.einsum("gtj,jd->tgd", torch.softmax(score.masked_fill(hidden, -math.inf), -1), v)
    return {"out": out.view(s["T"], -1)}


def _exact_tree(s):
    """Token by token, along its way to the root; the path step by step from the root."""
    q_start, pos0, parents, tokens, choice = _host(s, "q_start", "pos0", "parents", "tokens", "choice")
    words = _words(s)
    mask, pos = np.zeros((s["T"], words), np.int64), np.zeros(s["T"], np.int32)
    path, n_path, then = np.full((s["n"], s["new"]), -1, np.int32), np.zeros(s["n"], np.int32), np.zeros(s["n"], np.int32)
    for i in range(s["n"]):
        a, b = int(q_start[i]), int(q_start[i + 1])
        of, children = parents[a:b], {}
        for t in range(b - a):
            way = _walk(of, t)
            pos[a + t] = pos0[i] + len(way) - 1
            number = sum(1 << u for u in way)
            for w in range(words):
                word = number >> (64 * w) & (1 << 64) - 1
                mask[a + t, w] = word - (1 << 64) if word >> 63 else word
            children.setdefault(int(of[t]), []).append(t)
        at, steps = 0, [0]
        while True:
            agree = [u for u in children.get(at, []) if tokens[a + u] == choice[a + at]]
            if not agree:
                break
            at = agree[0]
            steps.append(at)
        path[i, :len(steps)], n_path[i], then[i] = steps, len(steps), choice[a + at]
    return {"mask": mask, "pos": pos, "path": path, "n_path": n_path, "next": then}


def _exact_keep(s):
    """Row by row, from copies of the pools as they were."""
    path, n_path, pos0, table, seq = _host(s, "path", "n_path", "pos0", "table", "seq")
    B, out = s["page"], {}
    for name in ("k_pool", "v_pool"):
        new = s[name].double()
        for i in range(s["n"]):
            for r in range(n_path[i]):
                to, at = int(pos0[i]) + r, int(pos0[i]) + int(path[i, r])
                new[:, int(table[seq[i], to // B]), :, to % B] = s[name][:, int(table[seq[i], at // B]), :, at % B].double()
        out[name] = new
    return out
