"""The attention operators' workloads, their plain forms and their exact values.

Four kinds of case:

    rope     per-head norm and rotation of queries and keys   (ops.qk_norm_rope)
    append   the same, with keys and values written to pages  (ops.kv_append)
    attend   attention over a paged cache                     (ops.paged_attention)
    prefix   the same for a batch that shares a long prefix   (ops.paged_attention, prefix_pages)

With `own` false, run() computes a case in elementary torch operations in 32
bits; with `own` true it makes the calls of warp_b200.ops.  Sizes are those of
this repository's stacks (hidden 2304 and 7168 as heads of 128 or 64, batch 32,
prompts of 512 tokens) and generic ones around them.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases --------------------------------------------------------------------------


def listed():
    return [
        # One token's queries and keys in a hidden-2304 layer: a call whose latency counts.
        {"name": "rope_token", "kind": "rope", "tokens": 1, "heads": 18, "kv_heads": 2, "dim": 128,
         "rot": 128, "interleaved": False, "norm": True, "scaling": "none", "far": 4000,
         "type": "f32", "out": "bf16"},
        # A long prompt's queries and keys, half of each head rotated, positions stretched eightfold.
        {"name": "rope_prompt", "kind": "rope", "tokens": 8191, "heads": 56, "kv_heads": 8,
         "dim": 128, "rot": 64, "interleaved": True, "norm": False, "scaling": "yarn",
         "far": 120000, "type": "bf16", "out": "bf16"},
        # A decode step of 32 streams: the fp32 projections of one layer into its cache.
        {"name": "append_step", "kind": "append", "batch": 32, "q_max": 1, "kv_max": 900,
         "heads": 56, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "norm": True,
         "scaling": "none", "page": 64, "heads_first": False, "type": "f32", "out": "bf16"},
        # Ragged prompts of a 64-wide head, a quarter rotated, pages of 16 laid out head by head.
        {"name": "append_prompts", "kind": "append", "batch": 5, "q_max": 1500, "kv_max": 1777,
         "heads": 36, "kv_heads": 4, "dim": 64, "rot": 16, "interleaved": True, "norm": False,
         "scaling": "linear", "page": 16, "heads_first": True, "type": "f16", "out": "f16"},
        # One prompt of 16 thousand tokens.
        {"name": "append_long", "kind": "append", "batch": 1, "q_max": 16384, "kv_max": 16384,
         "heads": 56, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "norm": True,
         "scaling": "yarn", "page": 128, "heads_first": False, "type": "bf16", "out": "bf16"},
        # One stream's next token over a short context: latency.
        {"name": "decode_one", "kind": "attend", "batch": 1, "q_max": 1, "kv_max": 777, "prefix": 0,
         "heads": 18, "kv_heads": 2, "dim": 128, "causal": True, "page": 16,
         "heads_first": False, "type": "bf16"},
        # 32 streams of unequal length, one of them without a key.
        {"name": "decode_batch", "kind": "attend", "batch": 32, "q_max": 1, "kv_max": 8192,
         "prefix": 0, "heads": 56, "kv_heads": 8, "dim": 128, "causal": True, "page": 64,
         "heads_first": False, "type": "bf16"},
        # Two streams of a long context: the keys have to be split over the card.
        {"name": "decode_long", "kind": "attend", "batch": 2, "q_max": 1, "kv_max": 131071,
         "prefix": 0, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "page": 32,
         "heads_first": True, "type": "f16"},
        # Chunks of 512 tokens and less that continue prompts already in the cache.
        {"name": "chunk", "kind": "attend", "batch": 3, "q_max": 512, "kv_max": 4500, "prefix": 0,
         "heads": 36, "kv_heads": 4, "dim": 64, "causal": True, "page": 16,
         "heads_first": False, "type": "bf16"},
        # A whole prompt at once.
        {"name": "prompt", "kind": "attend", "batch": 1, "q_max": 8192, "kv_max": 8192, "prefix": 0,
         "heads": 56, "kv_heads": 8, "dim": 128, "causal": True, "page": 64,
         "heads_first": False, "type": "bf16"},
        # A few streams behind a short instruction.
        {"name": "prefix_few", "kind": "prefix", "batch": 8, "q_max": 1, "kv_max": 65,
         "prefix": 515, "heads": 36, "kv_heads": 4, "dim": 64, "causal": True, "page": 16,
         "heads_first": False, "type": "f16"},
        # 64 streams that answer questions on one long document.
        {"name": "prefix_many", "kind": "prefix", "batch": 64, "q_max": 1, "kv_max": 1024,
         "prefix": 16001, "heads": 56, "kv_heads": 8, "dim": 128, "causal": True, "page": 64,
         "heads_first": False, "type": "bf16"},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    kind = rng.choice(["rope", "append", "attend", "attend", "prefix"])
    heads, kv_heads = rng.choice([(18, 2), (36, 4), (56, 8), (32, 8), (12, 12), (8, 1), (16, 1),
                                  (20, 4)])
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128])}
    if kind in ("rope", "append"):
        c["rot"] = rng.choice([c["dim"], c["dim"] // 2, c["dim"] // 4, c["dim"] - 12])
        c["interleaved"] = rng.random() < 0.5
        c["norm"] = rng.random() < 0.6
        c["scaling"] = rng.choice(["none", "linear", "ntk", "yarn"])
        c["type"] = rng.choice(["f32", "f16", "bf16"])
        c["out"] = c["type"] if c["type"] != "f32" else rng.choice(["f16", "bf16"])
    else:
        c["type"] = rng.choice(["f16", "bf16"])
    if kind == "rope":
        if c["type"] == "f32" and rng.random() < 0.5:
            c["out"] = "f32"
        c["tokens"] = log(1, 12000)
        c["far"] = log(64, 1000000)
        return c
    c["page"] = rng.choice([16, 32, 64, 128])
    c["heads_first"] = rng.random() < 0.3
    if kind == "append":
        c["batch"] = log(1, 64)
        c["q_max"] = log(1, 12000 // c["batch"])
        c["kv_max"] = c["q_max"] + log(1, 2000)
        return c
    c["causal"] = rng.random() < 0.8
    c["prefix"] = 0
    if kind == "prefix":
        c["batch"] = log(2, 96)
        c["prefix"] = log(64, 16000)
        c["q_max"] = rng.choice([1, 1, 1, 2, 5])
        c["kv_max"] = c["q_max"] + log(1, 1000)
        return c
    if rng.random() < 0.5:
        c["batch"] = log(1, 64)
        c["q_max"] = 1
        c["kv_max"] = log(1, min(131072, 262144 // c["batch"]))
    else:
        c["batch"] = log(1, 8)
        c["q_max"] = log(2, 3000 // c["batch"])
        c["kv_max"] = c["q_max"] + log(1, 6000 // c["batch"])
    return c


def _lengths(case):
    """Query and key counts of each request, by the case alone: unequal, the first the longest,
    and the second of more than eight single-token requests without a key."""
    batch, q_max, kv_max = case["batch"], case["q_max"], case["kv_max"]
    q, kv = [], []
    for i in range(batch):
        part = 1.0 - 0.8 * ((i * 0.6180339887) % 1.0)
        q.append(max(1, int(q_max * part)))
        kv.append(max(q[-1], int(kv_max * (1.0 - 0.8 * ((i * 0.4142135624) % 1.0)))))
    if batch > 8 and q_max == 1 and case["kind"] == "attend":
        kv[1] = 0
    return q, kv


def work(case):
    size = torch.empty(0, dtype=TYPES[case["type"]]).element_size()
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("rope", "append"):
        wide = torch.empty(0, dtype=TYPES[case["out"]]).element_size()
        append = case["kind"] == "append"
        tokens = sum(_lengths(case)[0]) if append else case["tokens"]
        values = tokens * (heads + (2 if append else 1) * kv_heads) * dim
        turned = tokens * (heads + kv_heads)
        return {"bytes": values * (size + wide) + tokens * (12 if append else 4),
                "flops": turned * (3 * case["rot"] + (4 * dim if case["norm"] else 0))}
    q, kv = _lengths(case)
    prefix = case["prefix"]
    pairs = sum(n * prefix for n in q)
    for n, length in zip(q, kv):
        if case["causal"]:
            first = length - n + 1
            pairs += sum(max(0, first + i) for i in range(n))
        else:
            pairs += n * length
    keys = prefix + sum(kv)
    return {"bytes": 2 * sum(q) * heads * dim * size + 2 * keys * kv_heads * dim * size,
            "flops": 4 * dim * heads * pairs}


# ---- inputs -------------------------------------------------------------------------


def _frequencies(case):
    """Radians a position of each rotated pair, in 64 bits, and the factor on cos and sin."""
    rot, base, factor, trained = case["rot"], 10000.0, 8.0, 16384
    i = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    if case["scaling"] == "ntk":
        base *= factor ** (rot / (rot - 2.0))
    f = base ** -i
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        def at(turns):
            return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(0, math.floor(at(32.0))), min(rot - 1, math.ceil(at(1.0)))
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rows(g, tokens, heads, kv_heads, dim, dtype, values):
    """Queries, keys and, where asked, values as a projection leaves them: parts of one row."""
    parts = heads + (2 if values else 1) * kv_heads
    x = torch.randn(tokens, parts, dim, generator=g, device="cuda") * 1.5
    x = x.to(dtype)
    return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]


def _pool(g, n, case, dtype):
    """Pages [n][page][kv_heads][dim] of keys or values, held head by head where the case says so."""
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    shape = (n, kv_heads, page, dim) if case["heads_first"] else (n, page, kv_heads, dim)
    x = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
    return x.transpose(1, 2) if case["heads_first"] else x


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    dtype = TYPES[case["type"]]
    s = {"case": case}
    if case["kind"] in ("rope", "append"):
        f, s["rot_scale"] = _frequencies(case)
        s["inv_freq"] = f.cuda()
        s["out"] = TYPES[case["out"]]
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"] = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda")
            s["k_norm"] = 1 + 0.1 * torch.randn(dim, generator=g, device="cuda")
    if case["kind"] == "rope":
        s["q"], s["k"], _ = _rows(g, case["tokens"], heads, kv_heads, dim, dtype, False)
        s["positions"] = torch.randint(0, case["far"], (case["tokens"],), generator=g,
                                       device="cuda", dtype=torch.int32)
        return s
    q_len, kv_len = _lengths(case)
    page, prefix = case["page"], case["prefix"] if case["kind"] == "prefix" else 0
    tokens, batch = sum(q_len), len(q_len)
    wide = max(1, -(-max(kv_len) // page))
    front = -(-prefix // page)
    count = batch * wide + front + 1
    order = torch.randperm(count, generator=g, device="cuda").int()
    s["pages"] = order[:batch * wide].view(batch, wide).contiguous()
    kept = s["out"] if case["kind"] == "append" else dtype
    s["k_pages"], s["v_pages"] = _pool(g, count, case, kept), _pool(g, count, case, kept)
    starts = [0]
    for n in q_len:
        starts.append(starts[-1] + n)
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    if case["kind"] == "append":
        s["q"], s["k"], s["v"] = _rows(g, tokens, heads, kv_heads, dim, dtype, True)
        request = torch.repeat_interleave(torch.arange(batch, device="cuda"),
                                          torch.tensor(q_len, device="cuda"))
        at = torch.arange(tokens, device="cuda") - s["q_start"][request].long()
        at += s["kv_len"][request].long() - torch.tensor(q_len, device="cuda")[request]
        s["positions"] = at.int()
        s["slots"] = s["pages"][request, at // page].long() * page + at % page
        return s
    s["prefix_pages"] = order[batch * wide:batch * wide + front].contiguous() if prefix else None
    s["prefix"], s["q_max"], s["kv_max"] = prefix, max(q_len), max(kv_len)
    # Queries wide enough that a row's weights are neither flat nor one key alone.
    s["q"] = (1.7 * torch.randn(tokens, heads, dim, generator=g, device="cuda")).to(dtype)
    return s


# ---- passes -------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        from warp_b200 import ops
        if kind == "rope":
            return ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"],
                                    q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6,
                                    interleaved=s["case"]["interleaved"],
                                    rot_scale=s["rot_scale"], out_dtype=s["out"])
        if kind == "append":
            q = ops.kv_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"],
                              s["positions"], s["inv_freq"], q_norm=s["q_norm"],
                              k_norm=s["k_norm"], eps=1e-6, interleaved=s["case"]["interleaved"],
                              rot_scale=s["rot_scale"])
            return q, s["k_pages"], s["v_pages"]
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["pages"], s["kv_len"],
                                   s["q_start"], max_q=s["q_max"], max_kv=s["kv_max"],
                                   causal=s["case"]["causal"], prefix_pages=s["prefix_pages"],
                                   prefix_len=s["prefix"])
    if kind == "rope":
        return _plain_rope(s, s["q"], s["q_norm"]), _plain_rope(s, s["k"], s["k_norm"])
    if kind == "append":
        page = s["case"]["page"]
        at, off = s["slots"] // page, s["slots"] % page
        q = _plain_rope(s, s["q"], s["q_norm"])
        s["k_pages"][at, off] = _plain_rope(s, s["k"], s["k_norm"])
        s["v_pages"][at, off] = s["v"].to(s["out"])
        return q, s["k_pages"], s["v_pages"]
    return _plain_attention(s)


def _plain_rope(s, x, w):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    # The angle is the one thing in 64 bits: a far position times a frequency has no
    # fraction of a turn left in 32.
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos = (torch.cos(angle).float() * s["rot_scale"])[:, None]
    sin = (torch.sin(angle).float() * s["rot_scale"])[:, None]
    rot = s["case"]["rot"]
    turned, rest = x[..., :rot], x[..., rot:]
    if s["case"]["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1).to(s["out"])


def _plain_attention(s):
    case, q = s["case"], s["q"]
    page, heads, kv_heads, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    group, batch, wide, longest = heads // kv_heads, case["batch"], s["q_max"], s["kv_max"]
    start, count = s["q_start"][:-1].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    i = torch.arange(wide, device="cuda")
    token = (start[:, None] + i).clamp(max=q.shape[0] - 1)
    # [batch][kv head][query * group][dim]
    x = q[token].float().view(batch, wide, kv_heads, group, dim).permute(0, 2, 1, 3, 4)
    x = x.reshape(batch, kv_heads, wide * group, dim) * (1.0 / math.sqrt(dim))
    j = torch.arange(longest, device="cuda")
    at = s["pages"][:, j // page].long()
    k = s["k_pages"][at, j % page].float().permute(0, 2, 3, 1)
    scores = x @ k
    seen = s["kv_len"].long()[:, None].expand(batch, wide)
    if case["causal"]:
        seen = torch.minimum(seen, seen - count[:, None] + i + 1)
    hidden = (j >= seen[..., None])[:, None, :, None]
    scores.view(batch, kv_heads, wide, group, longest).masked_fill_(hidden, -math.inf)
    if s["prefix"]:
        p = torch.arange(s["prefix"], device="cuda")
        at_p = s["prefix_pages"][p // page].long()
        front = s["k_pages"][at_p, p % page].float().permute(1, 2, 0)
        scores = torch.cat((x @ front, scores), -1)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weights.sum(-1, keepdim=True)
    v = s["v_pages"][at, j % page].float().transpose(1, 2)
    o = weights[..., s["prefix"]:] @ v
    if s["prefix"]:
        o = o + weights[..., :s["prefix"]] @ s["v_pages"][at_p, p % page].float().transpose(0, 1)
    o = o / torch.where(total == 0, 1.0, total)
    o = o.view(batch, kv_heads, wide, group, dim).transpose(1, 2).reshape(batch, wide, heads, dim)
    return o[i < count[:, None]].to(q.dtype)


# ---- the definition in 64 bits --------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return (_exact_rope(s, s["q"], s["q_norm"]), _exact_rope(s, s["k"], s["k_norm"]))
    if case["kind"] == "append":
        k, v = s["k_pages"].double(), s["v_pages"].double()
        page = case["page"]
        k[s["slots"] // page, s["slots"] % page] = _exact_rope(s, s["k"], s["k_norm"])
        v[s["slots"] // page, s["slots"] % page] = s["v"].double()
        return _exact_rope(s, s["q"], s["q_norm"]), k, v
    return _exact_attention(s)


def _exact_rope(s, x, w):
    """Each pair as a complex number times s * exp(i * position * frequency)."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
    half = s["inv_freq"].numel()
    by_pair = torch.arange(2 * half, device="cuda")
    by_pair = by_pair.view(half, 2) if s["case"]["interleaved"] else by_pair.view(2, half).t()
    turn = torch.polar(torch.full_like(s["inv_freq"], s["rot_scale"]).expand(x.shape[0], half),
                       s["positions"].double().outer(s["inv_freq"]))
    z = torch.view_as_complex(x[..., by_pair].contiguous()) * turn[:, None]
    y = x.clone()
    y[..., by_pair] = torch.view_as_real(z)
    return y


def _exact_attention(s):
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

    for head in range(case["kv_heads"]):
        mine = slice(head * group, (head + 1) * group)
        kp = vp = q.new_zeros(0, case["dim"])
        if s["prefix"]:
            kp = gathered(s["k_pages"], s["prefix_pages"], s["prefix"], head)
            vp = gathered(s["v_pages"], s["prefix_pages"], s["prefix"], head)
        for b, length in enumerate(lengths):
            n = starts[b + 1] - starts[b]
            k = torch.cat((kp, gathered(s["k_pages"], s["pages"][b], length, head)))
            v = torch.cat((vp, gathered(s["v_pages"], s["pages"][b], length, head)))
            if not len(k):
                continue
            x = torch.einsum("tgd,kd->tgk", q[starts[b]:starts[b + 1], mine], k)
            x = x / math.sqrt(case["dim"])
            if case["causal"]:
                key = torch.arange(len(k), device="cuda") - s["prefix"]
                query = torch.arange(n, device="cuda") + (length - n)
                x = x.masked_fill((key > query[:, None])[:, None], -math.inf)
            out[starts[b]:starts[b + 1], mine] = torch.einsum("tgk,kd->tgd", x.softmax(-1), v)
    return out
