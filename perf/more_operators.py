"""Workloads of a step of drafted tokens, their plain forms and their exact values.

Four kinds of case:

    plan     pages handed out, slots, positions and tree masks  (ops.step_plan)
    tree     attention of drafted trees over a paged cache      (ops.tree_attention)
    pick     penalties, biases and masks on logits, the choice  (ops.pick_tokens)
    accept   drafted tokens checked, their keys put in order    (ops.tree_accept)

With `own` false, run() computes a case in elementary torch operations; with `own` true
it makes the calls of warp_b200.ops.  Sizes are those of this repository's stacks
(hidden 2304 and 7168 as heads of 128 or 64) and generic ones around them.

A request's drafted tokens are the nodes of a tree: node 0 is the last token that is
certain, every other node's parent comes before it, and a node sees its ancestors and itself.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOKENS = 1 << 17                # drafted and picked tokens of `accept` are below this


# ---- cases --------------------------------------------------------------------------


def listed():
    return [
        # A decode step of 32 streams, a token each: a new page for one in 64.
        {"name": "plan_step", "kind": "plan", "batch": 32, "nodes": 1, "kv_max": 900, "page": 64,
         "branch": 1.0},
        # 48 streams with trees of up to 61 drafted tokens, small pages.
        {"name": "plan_trees", "kind": "plan", "batch": 48, "nodes": 61, "kv_max": 3001, "page": 16,
         "branch": 2.5},
        # Prompts of up to 16 thousand tokens come in, and leave again.
        {"name": "plan_prompts", "kind": "plan", "batch": 6, "nodes": 16384, "kv_max": 16384,
         "page": 16, "branch": 0.0},
        # One stream's tree over a short context: latency.
        {"name": "tree_one", "kind": "tree", "batch": 1, "nodes": 26, "kv_max": 777, "prefix": 0,
         "heads": 18, "kv_heads": 2, "dim": 128, "page": 16, "heads_first": False, "type": "bf16",
         "branch": 3.0},
        # 32 streams of unequal length, 16 drafted tokens and fewer each.
        {"name": "tree_batch", "kind": "tree", "batch": 32, "nodes": 16, "kv_max": 8192, "prefix": 0,
         "heads": 56, "kv_heads": 8, "dim": 128, "page": 64, "heads_first": False, "type": "bf16",
         "branch": 1.7},
        # Two streams of a long context with trees of 64.
        {"name": "tree_long", "kind": "tree", "batch": 2, "nodes": 64, "kv_max": 131071, "prefix": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "heads_first": True, "type": "f16",
         "branch": 2.0},
        # Streams behind one instruction, a chain of five drafted tokens and fewer each.
        {"name": "tree_prefix", "kind": "tree", "batch": 24, "nodes": 6, "kv_max": 500,
         "prefix": 4001, "heads": 36, "kv_heads": 4, "dim": 64, "page": 16, "heads_first": False,
         "type": "bf16", "branch": 1.0},
        # One stream's next token with the usual penalties: latency.
        {"name": "pick_one", "kind": "pick", "batch": 1, "nodes": 1, "vocab": 32000, "history": 700,
         "branch": 1.0, "penalties": True, "bias": "none", "masked": False, "keep": False,
         "type": "f32"},
        # Trees under a grammar: a mask for every node, and the adjusted logits kept for sampling.
        {"name": "pick_trees", "kind": "pick", "batch": 8, "nodes": 26, "vocab": 100003,
         "history": 8000, "branch": 3.0, "penalties": True, "bias": "none", "masked": True,
         "keep": True, "type": "bf16"},
        # 64 streams of 5 nodes and fewer over a large vocabulary, a bias for each stream.
        {"name": "pick_batch", "kind": "pick", "batch": 64, "nodes": 5, "vocab": 131072,
         "history": 30000, "branch": 1.0, "penalties": True, "bias": "each", "masked": False,
         "keep": False, "type": "f32"},
        # One stream's tree in the caches of 8 layers: latency.
        {"name": "accept_one", "kind": "accept", "batch": 1, "nodes": 26, "kv_max": 300,
         "layers": 8, "heads": 18, "kv_heads": 2, "dim": 128, "page": 16, "heads_first": False,
         "type": "bf16", "branch": 2.2},
        # 48 streams' trees in the caches of 32 layers.
        {"name": "accept_batch", "kind": "accept", "batch": 48, "nodes": 61, "kv_max": 160,
         "layers": 32, "heads": 56, "kv_heads": 8, "dim": 128, "page": 32, "heads_first": False,
         "type": "bf16", "branch": 1.6},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    kind = rng.choice(["plan", "tree", "tree", "pick", "accept"])
    c = {"kind": kind, "branch": rng.choice([1.0, 1.3, 2.0, 3.5])}
    if kind == "plan":
        c["page"] = rng.choice([16, 32, 64, 128])
        c["batch"] = log(1, 256)
        if rng.random() < 0.3:          # prompts: no tree
            c["branch"], c["nodes"] = 0.0, log(1, 48000 // c["batch"])
        else:
            c["nodes"] = log(1, min(200, 6000 // c["batch"]))
        c["kv_max"] = c["nodes"] + log(1, 16000)
        return c
    if kind == "pick":
        c["batch"] = log(1, 96)
        c["nodes"] = log(1, max(1, min(64, 300 // c["batch"])))
        c["vocab"] = log(1000, 160000)
        c["history"] = log(1, 30000)
        c["type"] = rng.choice(["f32", "f32", "f16", "bf16"])
        c["penalties"] = rng.random() < 0.8
        c["bias"] = rng.choice(["none", "all", "each"])
        c["masked"] = rng.random() < 0.5
        c["keep"] = rng.random() < 0.4
        if c["batch"] * c["nodes"] * c["vocab"] > 20_000_000:
            c["vocab"] = 20_000_000 // (c["batch"] * c["nodes"])
        return c
    c["heads"], c["kv_heads"] = rng.choice([(18, 2), (36, 4), (56, 8), (32, 8), (12, 12), (8, 1),
                                            (16, 1), (20, 4)])
    c["dim"] = rng.choice([64, 128])
    c["type"] = rng.choice(["f16", "bf16"])
    c["page"] = rng.choice([16, 32, 64, 128])
    c["heads_first"] = rng.random() < 0.3
    if kind == "accept":
        c["batch"] = log(1, 64)
        c["nodes"] = log(2, 90)
        c["kv_max"] = c["nodes"] + log(1, 200)
        c["layers"] = log(1, 64)
        size = c["batch"] * (c["kv_max"] + c["page"]) * c["layers"] * c["kv_heads"] * c["dim"]
        if size > 400_000_000:
            c["layers"] = max(1, c["layers"] * 400_000_000 // size)
        return c
    c["batch"] = log(1, 48)
    c["nodes"] = log(1, min(300, 1500 // c["batch"]))
    most = 400_000_000 // (c["batch"] * c["nodes"] * c["heads"])
    c["prefix"] = min(log(64, 8000), most // 2) if rng.random() < 0.25 else 0
    most -= c["prefix"]
    c["kv_max"] = c["nodes"] + log(1, max(1, min(100000, 200000 // c["batch"], most)))
    return c


def _lengths(case):
    """Nodes and keys of each request, the nodes counted, by the case alone: unequal, the first
    the longest."""
    nodes, kv = [], []
    for i in range(case["batch"]):
        part = 1.0 - 0.8 * ((i * 0.6180339887) % 1.0)
        nodes.append(max(1, int(case["nodes"] * part)))
        if "kv_max" in case:
            kv.append(max(nodes[-1], int(case["kv_max"] * (1.0 - 0.8 * ((i * 0.4142135624) % 1.0)))))
    return nodes, kv


def _parents(case, n):
    """Parents of n nodes in order of their depth: a chain where `branch` is 1, else about so
    many children each."""
    return [-1] + [int((i - 1) / case["branch"]) for i in range(1, n)]


def _ancestors(case, n):
    """The nodes that each of n nodes sees, ascending."""
    paths = []
    for i, p in enumerate(_parents(case, n)):
        paths.append((paths[p] if p >= 0 else []) + [i])
    return paths


def _accepted(case, n, b):
    """The path of request b that is accepted, by the case alone.  Keys that move come from
    behind every place they move to, so that a pass can be repeated on the same caches."""
    def repeatable(path):
        moved = {d for d, i in enumerate(path) if d != i}
        return not moved & {path[d] for d in moved}
    good = [p for p in _ancestors(case, n) if repeatable(p)]
    most = max(len(p) for p in good)
    good = [p for p in good if len(p) >= min(most, 4 + b % 4)]
    return good[(7 * b + 3) % len(good)]


def work(case):
    nodes, kv = _lengths(case)
    tokens, batch = sum(nodes), case["batch"]
    if case["kind"] == "plan":
        page, tree = case["page"], case["branch"] > 0
        moved = sum(-(-k // page) - -(-(k - n) // page) for n, k in zip(nodes, kv))
        words = -(-max(nodes) // 64) if tree else 0
        # two calls: what a step takes is given back after it
        return {"bytes": tokens * (12 + (4 + 8 * words if tree else 0)) + 2 * (12 * batch + 8 * moved),
                "flops": 0}
    if case["kind"] == "pick":
        size = torch.empty(0, dtype=TYPES[case["type"]]).element_size()
        vocab = case["vocab"]
        bias = {"none": 0, "all": 1, "each": batch}[case["bias"]]
        return {"bytes": tokens * vocab * size * (2 if case["keep"] else 1) + bias * vocab * 4 +
                (tokens * -(-vocab // 32) * 4 if case["masked"] else 0) +
                (batch * case["history"] * 4 if case["penalties"] else 0) + tokens * 4,
                "flops": tokens * vocab * (1 + (bias > 0))}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "accept":
        moved = sum(sum(d != i for d, i in enumerate(_accepted(case, n, b)))
                    for b, n in enumerate(nodes))
        words = -(-max(nodes) // 64)
        return {"bytes": 2 * moved * case["layers"] * 2 * kv_heads * dim * 2 +
                tokens * (8 + 8 * words) + batch * (12 + 8 * max(nodes)), "flops": 0}
    pairs = sum(n * (k - n + case["prefix"]) + sum(len(p) for p in _ancestors(case, n))
                for n, k in zip(nodes, kv))
    keys = case["prefix"] + sum(kv)
    return {"bytes": 4 * tokens * heads * dim + 4 * keys * kv_heads * dim +
            8 * tokens * -(-max(nodes) // 64), "flops": 4 * dim * heads * pairs}


# ---- inputs -------------------------------------------------------------------------


def _starts(lengths):
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32, device="cuda")


def _seen(case, nodes):
    """[tokens][words] int64: bit m of a token's words says that it sees node m of its request."""
    words, rows = -(-max(nodes) // 64), []
    for n in nodes:
        bits = []
        for i, p in enumerate(_parents(case, n)):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        rows += [b.to_bytes(8 * words, "little") for b in bits]
    return torch.frombuffer(bytearray(b"".join(rows)), dtype=torch.int64).view(-1, words).cuda()


def _pool_of_pages(g, n, case):
    """Keys or values [n][page][kv_heads][dim], held head by head where the case says so."""
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    shape = (n, kv_heads, page, dim) if case["heads_first"] else (n, page, kv_heads, dim)
    x = torch.randn(shape, generator=g, device="cuda", dtype=TYPES[case["type"]])
    return x.transpose(1, 2) if case["heads_first"] else x


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    nodes, kv = _lengths(case)
    tokens, batch = sum(nodes), len(nodes)
    s = {"case": case, "tokens": tokens, "max_q": max(nodes), "q_start": _starts(nodes),
         "kv_len": torch.tensor(kv or [0], dtype=torch.int32, device="cuda")}
    if case["kind"] == "plan":
        page = case["page"]
        s["wide"] = wide = -(-max(kv) // page)
        before = [k - n for n, k in zip(nodes, kv)]
        s["before"] = torch.tensor(before, dtype=torch.int32, device="cuda")
        s["no_tokens"] = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
        held = [-(-n // page) for n in before]
        s["held"] = torch.tensor(held, dtype=torch.int32, device="cuda")
        total = sum(-(-k // page) for k in kv) + 5
        order = torch.randperm(total, generator=g, device="cuda").int()
        has = torch.arange(wide, device="cuda") < s["held"][:, None]
        s["pages"] = torch.full((batch, wide), -1, dtype=torch.int32, device="cuda")
        s["pages"][has] = order[:sum(held)]
        s["pool"] = torch.zeros(1 + total, dtype=torch.int32, device="cuda")
        s["pool"][0] = total - sum(held)
        s["pool"][1:1 + total - sum(held)] = order[sum(held):]
        s["parents"] = None
        if case["branch"] > 0:
            s["parents"] = torch.tensor([p for n in nodes for p in _parents(case, n)],
                                        dtype=torch.int32, device="cuda")
        return s
    if case["kind"] == "pick":
        return _prepare_pick(s, case, g, nodes)
    page = case["page"]
    s["seen"] = _seen(case, nodes)
    prefix = case.get("prefix", 0)
    wide, front = -(-max(kv) // page), -(-prefix // page)
    count = batch * wide + front + 1
    order = torch.randperm(count, generator=g, device="cuda").int()
    s["pages"] = order[:batch * wide].view(batch, wide).contiguous()
    s["kv_max"], s["prefix"] = max(kv), prefix
    if case["kind"] == "tree":
        s["prefix_pages"] = order[batch * wide:batch * wide + front].contiguous() if prefix else None
        s["k_pages"], s["v_pages"] = _pool_of_pages(g, count, case), _pool_of_pages(g, count, case)
        # Queries wide enough that a row's weights are neither flat nor one key alone.
        s["q"] = (1.7 * torch.randn(tokens, case["heads"], case["dim"], generator=g,
                                    device="cuda")).to(TYPES[case["type"]])
        return s
    # [layer][keys, values][pages]...
    x = _pool_of_pages(g, 2 * case["layers"] * count, case)
    s["pools"] = x.unflatten(0, (case["layers"], 2, count))
    s["caches"] = [(c[0], c[1]) for c in s["pools"].unbind()]
    drafted = torch.randint(0, TOKENS, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    picked = torch.randint(0, TOKENS, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    start, ups, downs = 0, [], []
    for b, n in enumerate(nodes):
        path = _accepted(case, n, b)
        ups += [start + i for i in path[:-1]]
        downs += [start + i for i in path[1:]]
        start += n
    picked[torch.tensor(ups, dtype=torch.long, device="cuda")] = \
        drafted[torch.tensor(downs, dtype=torch.long, device="cuda")]
    s["drafted"], s["picked"] = drafted, picked
    return s


def _prepare_pick(s, case, g, nodes):
    vocab, batch, tokens = case["vocab"], case["batch"], s["tokens"]
    s["seen"] = _seen(case, nodes)
    s["logits"] = (3 * torch.randn(tokens, vocab, generator=g, device="cuda")).to(TYPES[case["type"]])

    def usual(*shape):          # few tokens make up most of a text
        u = torch.rand(shape, generator=g, device="cuda")
        return (vocab * u ** 4).int().clamp(max=vocab - 1)
    s["drafted"] = usual(tokens)
    for name in ("history", "history_len", "repetition", "frequency", "presence", "bias", "allowed"):
        s[name] = None
    if case["penalties"]:
        s["history"] = usual(batch, case["history"])
        part = torch.arange(batch, device="cuda") * 0.7548776662 % 1.0
        s["history_len"] = (case["history"] * (1 - 0.9 * part)).int()
        s["repetition"] = 1 + 0.5 * torch.rand(batch, generator=g, device="cuda")
        s["frequency"] = 0.3 * torch.rand(batch, generator=g, device="cuda")
        s["presence"] = torch.rand(batch, generator=g, device="cuda")
    if case["bias"] != "none":
        shape = (batch, vocab) if case["bias"] == "each" else (vocab,)
        s["bias"] = torch.randn(shape, generator=g, device="cuda")
    if case["masked"]:
        shape = (tokens, -(-vocab // 32))
        a, b = (torch.randint(-2 ** 31, 2 ** 31, shape, generator=g, device="cuda",
                              dtype=torch.int64).int() for _ in range(2))
        s["allowed"] = a & b    # a quarter of the tokens
        s["allowed"][tokens // 2] = 0       # a node behind the grammar's end: nothing
    s["out"] = torch.empty_like(s["logits"]) if case["keep"] else None
    return s


# ---- passes -------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        from warp_b200 import ops
        if kind == "plan":
            planned = ops.step_plan(s["q_start"], s["kv_len"], s["pages"], s["case"]["page"],
                                    s["tokens"], held=s["held"], pool=s["pool"],
                                    parents=s["parents"], max_q=s["max_q"])
            # the requests go back to where they were
            ops.step_plan(s["no_tokens"], s["before"], s["pages"], s["case"]["page"], 0,
                          held=s["held"], pool=s["pool"])
            return *planned, s["pages"], s["held"], s["pool"]
        if kind == "tree":
            return ops.tree_attention(s["q"], s["k_pages"], s["v_pages"], s["pages"], s["kv_len"],
                                      s["q_start"], s["seen"], max_q=s["max_q"],
                                      max_kv=s["kv_max"], prefix_pages=s["prefix_pages"],
                                      prefix_len=s["prefix"])
        if kind == "pick":
            picked = ops.pick_tokens(s["logits"], s["q_start"], history=s["history"],
                                     history_len=s["history_len"], repetition=s["repetition"],
                                     frequency=s["frequency"], presence=s["presence"],
                                     bias=s["bias"], allowed=s["allowed"], drafted=s["drafted"],
                                     seen=s["seen"], out=s["out"])
            return picked if s["out"] is None else (picked, s["out"])
        done = ops.tree_accept(s["drafted"], s["picked"], s["seen"], s["q_start"], s["kv_len"],
                               s["max_q"], caches=s["caches"], pages=s["pages"])
        return *done, s["pools"]
    if kind == "plan":
        planned = _plain_plan(s)
        _plain_pages(s, s["before"])
        return *planned, s["pages"], s["held"], s["pool"]
    if kind == "tree":
        return _plain_tree(s)
    if kind == "pick":
        return _plain_pick(s)
    return _plain_accept(s)


def _plain_pages(s, kv_len):
    """Gives back the pages that lengths do not need, then hands out those that they do."""
    page, wide, pool, pages = s["case"]["page"], s["wide"], s["pool"], s["pages"]
    entry = torch.arange(wide, device="cuda")
    need, had = (kv_len + page - 1) // page, s["held"]
    # the last entry of the last request first, so that they come off again in order
    give = (entry >= need[:, None]) & (entry < had[:, None])
    rank = give.sum() - give.flatten().cumsum(0).view_as(give)
    at = torch.where(give, pool[0] + rank + 1, pool.numel())
    more = torch.cat((pool, pool[:1]))
    more.scatter_(0, at.flatten(), pages.flatten())
    pool.copy_(more[:-1])
    pages.masked_fill_(give, -1)
    top = pool[0] + give.sum()
    take = (entry >= had[:, None]) & (entry < need[:, None])
    rank = take.flatten().cumsum(0).view_as(take) - 1
    got = take & (rank < top)
    pages.copy_(torch.where(got, pool[(top - rank).clamp(1, pool.numel() - 1)], pages))
    s["held"].copy_(torch.minimum(need, had) + got.sum(1))
    pool[0] = top - got.sum()


def _plain_plan(s):
    _plain_pages(s, s["kv_len"])
    page, t = s["case"]["page"], torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["q_start"], t.int(), right=True) - 1
    end = s["q_start"][b + 1]
    own_key = s["kv_len"][b] - end + t
    slots = s["pages"][b, own_key // page].long() * page + own_key % page
    if s["parents"] is None:
        return own_key.int(), slots
    # who sees whom within a request, doubled until the whole way up is in it
    n, first = s["max_q"], s["q_start"][b].long()
    node = torch.arange(n, device="cuda")
    sees = torch.zeros(s["case"]["batch"], n, n, device="cuda")
    sees[b, t - first] = ((node == (t - first)[:, None]) | (node == s["parents"][:, None])).float()
    for _ in range((n - 1).bit_length()):
        sees = (sees @ sees > 0).float()
    sees = sees[b, t - first]
    words = -(-n // 64)
    wide = torch.zeros(s["tokens"], words * 64, dtype=torch.int64, device="cuda")
    wide[:, :n] = sees
    seen = (wide.view(-1, words, 64) << torch.arange(64, device="cuda")).sum(-1)
    return (s["kv_len"][b] - end + first + sees.sum(1) - 1).int(), slots, seen


def _plain_tree(s):
    case, q = s["case"], s["q"]
    page, heads, kv_heads, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    group, batch, wide, longest = heads // kv_heads, case["batch"], s["max_q"], s["kv_max"]
    start, count = s["q_start"][:-1].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    i = torch.arange(wide, device="cuda")
    token = (start[:, None] + i).clamp(max=q.shape[0] - 1)
    # [batch][kv head][node * group][dim]
    x = q[token].float().view(batch, wide, kv_heads, group, dim).permute(0, 2, 1, 3, 4)
    x = x.reshape(batch, kv_heads, wide * group, dim) * (1.0 / math.sqrt(dim))
    j = torch.arange(longest, device="cuda")
    at = s["pages"][:, j // page].long()
    scores = x @ s["k_pages"][at, j % page].float().permute(0, 2, 3, 1)
    # the request's own nodes are its last keys
    node = j - (s["kv_len"].long() - count)[:, None]
    bits = s["seen"][token].gather(2, (node.clamp(0, wide - 1) // 64)[:, None].expand(-1, wide, -1))
    shown = (node < 0)[:, None] | ((bits >> (node.clamp(min=0) % 64)[:, None]) & 1).bool()
    shown &= (node < count[:, None])[:, None]
    scores.view(batch, kv_heads, wide, group, longest).masked_fill_(~shown[:, None, :, None],
                                                                    -math.inf)
    if s["prefix"]:
        p = torch.arange(s["prefix"], device="cuda")
        at_p = s["prefix_pages"][p // page].long()
        scores = torch.cat((x @ s["k_pages"][at_p, p % page].float().permute(1, 2, 0), scores), -1)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weights.sum(-1, keepdim=True)
    o = weights[..., s["prefix"]:] @ s["v_pages"][at, j % page].float().transpose(1, 2)
    if s["prefix"]:
        front = s["v_pages"][at_p, p % page].float().transpose(0, 1)
        o = o + weights[..., :s["prefix"]] @ front
    o = o / torch.where(total == 0, 1.0, total)
    o = o.view(batch, kv_heads, wide, group, dim).transpose(1, 2).reshape(batch, wide, heads, dim)
    return o[i < count[:, None]].to(q.dtype)


def _plain_pick(s):
    x = s["logits"].float()
    tokens, vocab = x.shape
    t = torch.arange(tokens, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["q_start"], t, right=True) - 1
    if s["history"] is not None:
        held = torch.arange(s["history"].shape[1], device="cuda") < s["history_len"][:, None]
        counts = torch.zeros(len(s["history"]), vocab, device="cuda")
        counts.scatter_add_(1, s["history"].long(), held.float())
        counts = counts[b]
        node = torch.arange(s["max_q"], device="cuda")
        sees = (s["seen"][:, node // 64] >> (node % 64)) & 1
        at = (s["q_start"][b].long()[:, None] + node).clamp(max=tokens - 1)
        counts.scatter_add_(1, s["drafted"][at].long(), sees.float())
        r, f, p = (s[k][b][:, None] for k in ("repetition", "frequency", "presence"))
        less = torch.where(x > 0, x / r, x * r) - f * counts - p
        x = torch.where(counts > 0, less, x)
    if s["bias"] is not None:
        x = x + (s["bias"][b] if s["bias"].dim() == 2 else s["bias"])
    if s["allowed"] is not None:
        v = torch.arange(vocab, device="cuda")
        x = torch.where((s["allowed"][:, v // 32] >> (v % 32).int()) & 1 == 1, x, -math.inf)
    top, picked = torch.where(x.isnan(), -math.inf, x).max(-1)
    first = (x == top[:, None]).int().argmax(-1)
    picked = torch.where(top == -math.inf, -1, first).int()
    if s["out"] is None:
        return picked
    s["out"].copy_(x)
    return picked, s["out"]


def _plain_accept(s):
    n, tokens = s["max_q"], s["tokens"]
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(s["q_start"], t.int(), right=True) - 1
    first = s["q_start"][b].long()
    node = torch.arange(n, device="cuda")
    sees = ((s["seen"][:, node // 64] >> (node % 64)) & 1).bool()
    local = (t - first)[:, None]
    parent = torch.where(sees & (node < local), node, -1).amax(1)
    fits = s["drafted"] == s["picked"][first + parent.clamp(min=0)]
    agrees = (local[:, 0] == 0) | ((parent >= 0) & fits & (s["drafted"] >= 0))
    at = (first[:, None] + node).clamp(max=tokens - 1)
    whole = sees[:, 0] & (agrees[at] | ~sees).all(1)
    # the longest path, the first of equal ones
    score = torch.where(whole, sees.sum(1) * (n + 1) + n - local[:, 0], -1)
    batch = len(s["q_start"]) - 1
    board = torch.full((batch, n), -1, device="cuda")
    board[b, local[:, 0]] = score
    best = s["q_start"][:-1].long() + board.argmax(1)
    on = sees[best]
    count = on.sum(1)
    order = torch.where(on, node, n).sort(1).values
    path = torch.where(node < count[:, None], order, -1)
    src = (s["q_start"][:-1].long()[:, None] + path.clamp(min=0))
    chosen = torch.where(path >= 0, s["picked"][src], -1)
    nodes = (s["q_start"][1:] - s["q_start"][:-1])
    base = (s["kv_len"] - nodes).long()
    # keys of the path to the places right behind the certain ones
    page = s["case"]["page"]
    which, d = (path > node).nonzero(as_tuple=True)
    now, then = base[which] + path[which, d], base[which] + d
    kept = s["pools"][:, :, s["pages"][which, now // page].long(), now % page]
    s["pools"][:, :, s["pages"][which, then // page].long(), then % page] = kept
    return (count.int(), path.int(), chosen.int(), (s["kv_len"] - nodes + count).int(), s["pools"])


# ---- the definition in 64 bits --------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "tree": _exact_tree, "pick": _exact_pick,
            "accept": _exact_accept}[case["kind"]](s)


def _exact_plan(s):
    """Request by request and page by page; the step's pages are given back at the end, so the
    table, the lengths and the pool are what they were."""
    case = s["case"]
    page, lengths, starts = case["page"], s["kv_len"].tolist(), s["q_start"].tolist()
    table, pool = s["pages"].tolist(), s["pool"].tolist()
    free = pool[1:1 + pool[0]]
    positions, slots, seen = [], [], []
    for b, length in enumerate(lengths):
        row = [p for p in table[b] if p >= 0]
        while len(row) * page < length:
            row.append(free.pop())
        n = starts[b + 1] - starts[b]
        for i, path in enumerate(_ancestors(case, n) if s["parents"] is not None else [()] * n):
            j = length - n + i
            slots.append(row[j // page] * page + j % page)
            positions.append(length - n + len(path) - 1 if path else j)
            word = [0] * -(-s["max_q"] // 64)
            for m in path:
                word[m // 64] |= 1 << m % 64
            seen.append([w - (1 << 64) if w >> 63 else w for w in word])
    made = [torch.tensor(positions, dtype=torch.int32), torch.tensor(slots)]
    if s["parents"] is not None:
        made.append(torch.tensor(seen))
    return *made, s["pages"], s["held"], s["pool"]


def _exact_tree(s):
    case = s["case"]
    q, page, group = s["q"].double(), case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    starts, lengths = s["q_start"].tolist(), s["kv_len"].tolist()
    if sum((b - a) * (n + s["prefix"]) for a, b, n in zip(starts, starts[1:], lengths)) \
            * case["heads"] * case["dim"] > 1e12:
        return None

    def gathered(pool, table, count, head):
        n = torch.arange(count, device="cuda")
        return pool[table[n // page].long(), n % page, head].double()

    for b, length in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        hidden = torch.ones(n, n, dtype=torch.bool)
        for i, path in enumerate(_ancestors(case, n)):
            hidden[i, path] = False
        hidden = torch.cat((torch.zeros(n, s["prefix"] + length - n, dtype=torch.bool), hidden), 1)
        hidden = hidden[:, None].cuda()
        for head in range(case["kv_heads"]):
            k, v = (gathered(x, s["pages"][b], length, head) for x in (s["k_pages"], s["v_pages"]))
            if s["prefix"]:
                k = torch.cat((gathered(s["k_pages"], s["prefix_pages"], s["prefix"], head), k))
                v = torch.cat((gathered(s["v_pages"], s["prefix_pages"], s["prefix"], head), v))
            mine = slice(head * group, (head + 1) * group)
            x = torch.einsum("tgd,kd->tgk", q[starts[b]:starts[b + 1], mine], k)
            x = (x / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
            out[starts[b]:starts[b + 1], mine] = torch.einsum("tgk,kd->tgd", x.softmax(-1), v)
    return out


def _exact_pick(s):
    case, starts = s["case"], s["q_start"].tolist()
    vocab, picked, rows = case["vocab"], [], []
    for b in range(case["batch"]):
        n = starts[b + 1] - starts[b]
        paths = _ancestors(case, n)
        before = None
        if s["history"] is not None:
            past = s["history"][b, :int(s["history_len"][b])].long()
            before = torch.bincount(past, minlength=vocab)
            rep, freq, pres = (float(s[k][b]) for k in ("repetition", "frequency", "presence"))
        for i in range(n):
            x = s["logits"][starts[b] + i].double()
            if before is not None:
                path = torch.tensor(paths[i], device="cuda") + starts[b]
                count = before + torch.bincount(s["drafted"][path].long(), minlength=vocab)
                hit = count > 0
                y = x[hit]
                x[hit] = y * rep ** (1 - 2 * (y > 0).double()) - freq * count[hit] - pres
            if s["bias"] is not None:
                x += (s["bias"][b] if case["bias"] == "each" else s["bias"]).double()
            if s["allowed"] is not None:
                word = s["allowed"][starts[b] + i].long()[:, None] >> torch.arange(32, device="cuda")
                x[(word & 1).flatten()[:vocab] == 0] = -math.inf
            best = x.max()
            picked.append(-1 if best == -math.inf else int((x == best).nonzero()[0]))
            if case["keep"]:
                rows.append(x)
    picked = torch.tensor(picked, dtype=torch.int32)
    return (picked, torch.stack(rows)) if case["keep"] else picked


def _exact_accept(s):
    """Node by node from the root: the longest of the paths whose tokens were picked."""
    case, page, n_max = s["case"], s["case"]["page"], s["max_q"]
    starts, lengths, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["pages"].tolist()
    drafted, picked = s["drafted"].tolist(), s["picked"].tolist()
    pools = s["pools"].double()
    count, path, chosen, after = [], [], [], []
    for b, length in enumerate(lengths):
        t0, n = starts[b], starts[b + 1] - starts[b]
        parents, best, reached = _parents(case, n), [0], {0: [0]}
        for i in range(1, n):
            up = reached.get(parents[i])
            if up and drafted[t0 + i] == picked[t0 + parents[i]]:
                reached[i] = up + [i]
                best = reached[i] if len(reached[i]) > len(best) else best
        for d, i in enumerate(best):
            now, then = length - n + i, length - n + d
            pools[:, :, table[b][then // page], then % page] = \
                pools[:, :, table[b][now // page], now % page].clone()
        rest = [-1] * (n_max - len(best))
        count.append(len(best))
        path.append(best + rest)
        chosen.append([picked[t0 + i] for i in best] + rest)
        after.append(length - n + len(best))
    return *(torch.tensor(x, dtype=torch.int32) for x in (count, path, chosen, after)), pools
