"""Cases of the paged-cache serving operators: what they compute, in plain torch and through the framework.

Four operators that a server of a Qwen2-like decoder runs around its linears:

* ``append``: rotary positions on the new queries and keys, the new keys and
  values written into the pages of their sequences;
* ``attention``: the new tokens' queries against their sequences' pages
  (causal: token i of n sees the keys up to its own), from one token per
  sequence to whole prompts;
* ``prefix``: the same where all sequences begin with one shared, already
  cached prefix, whose keys are read once for the batch;
* ``verify``: drafted tokens accepted or refused against the target's
  probabilities from given uniform numbers, and the token that follows.

A case is a dict of plain values. The batch's lengths follow from the case
alone; the values in the tensors follow from the seed.
"""

import functools
import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@functools.lru_cache(maxsize=None)
def _framework():
    return importlib.import_module("qwen2-int4-systems_b200")


# -- the cases ------------------------------------------------------------------

def listed():
    qwen = {"q_heads": 12, "kv_heads": 2, "head_dim": 128, "dtype": "bf16"}
    return [
        # A decode step of 64 sequences: one new token each, Qwen2-1.5B's heads (the serving workload's batch).
        {"name": "append: 64 decode steps", "op": "append", "batch": 64, "tokens": 1, "past": 1279, "ragged": False,
         "page": 16, "rot": 128, "interleaved": False, **qwen},
        # A scheduler's step over prompts of mixed lengths; rotary pairs side by side on part of the head.
        {"name": "append: ragged prompts", "op": "append", "batch": 13, "tokens": 4001, "past": 700, "ragged": True,
         "page": 32, "rot": 64, "interleaved": True, "q_heads": 16, "kv_heads": 4, "head_dim": 128, "dtype": "f16"},
        # Batch-1 decode behind a 512-token prompt (the single-stream workload).
        {"name": "attention: 1 sequence", "op": "attention", "batch": 1, "tokens": 1, "past": 640, "ragged": False,
         "page": 16, **qwen},
        # Batch-64 decode behind 1024-token prompts (the serving workload).
        {"name": "attention: 64 sequences", "op": "attention", "batch": 64, "tokens": 1, "past": 1150, "ragged": False,
         "page": 16, **qwen},
        # Drafts of five tokens checked for sequences of very different lengths, smaller heads, FP16.
        {"name": "attention: drafts", "op": "attention", "batch": 24, "tokens": 5, "past": 6000, "ragged": True,
         "page": 32, "q_heads": 16, "kv_heads": 4, "head_dim": 64, "dtype": "f16"},
        # One sequence with a long document behind it.
        {"name": "attention: long context", "op": "attention", "batch": 1, "tokens": 1, "past": 131001,
         "ragged": False, "page": 64, **qwen},
        # Chunks of prompts, some with keys cached by earlier chunks.
        {"name": "attention: prompt chunks", "op": "attention", "batch": 6, "tokens": 2047, "past": 3001,
         "ragged": True, "page": 16, **qwen},
        # One whole prompt.
        {"name": "attention: 8192-token prompt", "op": "attention", "batch": 1, "tokens": 8192, "past": 0,
         "ragged": False, "page": 16, **qwen},
        # A few sequences behind one short system prompt that ends inside a page's tile.
        {"name": "prefix: 8 on 1000 keys", "op": "prefix", "batch": 8, "tokens": 1, "past": 90, "ragged": True,
         "prefix": 1000, "page": 16, **qwen},
        # A full decode batch behind one long shared context.
        {"name": "prefix: 64 on 16384 keys", "op": "prefix", "batch": 64, "tokens": 1, "past": 511, "ragged": True,
         "prefix": 16384, "page": 64, **qwen},
        # One stream's four drafted tokens, the full vocabulary.
        {"name": "verify: 1 sequence", "op": "verify", "batch": 1, "drafts": 4, "vocab": 151936, "ragged": False},
        # A batch's drafts of different lengths.
        {"name": "verify: 64 sequences", "op": "verify", "batch": 64, "drafts": 5, "vocab": 151936, "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "prefix", "verify"))
    if op == "verify":
        vocab = _log(rng, 32000, 151936)
        return {"op": op, "batch": _log(rng, 1, 64), "drafts": rng.randint(1, 6), "vocab": vocab,
                "ragged": rng.random() < 0.5}
    kv_heads, group, head_dim = rng.choice(((2, 6, 128), (4, 4, 128), (8, 1, 128), (4, 4, 64), (2, 7, 64), (1, 8, 128)))
    case = {"op": op, "ragged": rng.random() < 0.6, "page": rng.choice((16, 32, 64)), "q_heads": kv_heads * group,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": rng.choice(("bf16", "f16"))}
    if op == "append":
        tokens = rng.choice((1, _log(rng, 2, 4000)))
        batch = _log(rng, 1, max(2, min(256, 30000 // tokens)))
        return {**case, "batch": batch, "tokens": tokens, "past": _log(rng, 1, 4000 if batch < 16 else 1500),
                "rot": rng.choice((head_dim, head_dim // 2)), "interleaved": rng.random() < 0.5}
    tokens = rng.choice((1, 1, rng.randint(2, 8), _log(rng, 9, 2000)))
    if op == "prefix":
        tokens = min(tokens, 8)
        return {**case, "batch": _log(rng, 2, 64), "tokens": tokens, "past": _log(rng, 1, 600),
                "prefix": _log(rng, 100, 16384 // tokens)}
    past = _log(rng, 1, 60000)
    most = min(64, 300000 // (past + tokens), int(5e8 / case["q_heads"] / tokens / (past + tokens)))
    return {**case, "batch": _log(rng, 1, max(2, most)), "tokens": tokens, "past": past}


# -- the batch's lengths, from the case alone ---------------------------------------

def _lengths(case):
    """(new tokens, keys cached before them) of each sequence. In a ragged batch they differ, and from four
    sequences on the second has no new token and the third nothing cached."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    batch, most, past = case["batch"], case["tokens"], case["past"]
    if not case["ragged"]:
        return [most] * batch, [past] * batch
    new = [rng.randint(max(1, most // 3), most) for _ in range(batch)]
    old = [int(past * rng.random() ** 1.5) for _ in range(batch)]
    new[0], old[-1] = most, past
    if batch >= 4:
        new[1], old[2] = 0, 0
    return new, old


def _drafted(case):
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if not case["ragged"]:
        return [case["drafts"]] * case["batch"]
    return [rng.randint(0, case["drafts"]) for _ in range(case["batch"])]


def _pairs(n, m):
    """Visible (query, key) pairs of n new tokens behind m cached keys."""
    return n * m + n * (n + 1) // 2


def work(case):
    if case["op"] == "verify":
        # The target's row for the token that follows, the draft's row too where one was refused (about four in
        # five of the drafts are accepted), the drafted tokens' own probabilities.
        v, some = case["vocab"], _drafted(case)
        rows = sum(2 - 0.8 ** k for k in some)
        return {"bytes": rows * v * 4 + sum(8 * k + 8 * k + 4 * k + 12 for k in some) + 8 * case["batch"] * (
            case["drafts"] + 1), "flops": 3 * rows * v}
    new, old = _lengths(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    total = sum(new)
    if case["op"] == "append":
        return {"bytes": total * ((hq + 2 * hk) * d * 2 * 2 + case["rot"] * 4), "flops": total * (hq + hk) * case["rot"] * 3}
    shared = case.get("prefix", 0)
    keys = shared + sum(n + m for n, m in zip(new, old) if n)
    pairs = sum(_pairs(n, m + shared) for n, m in zip(new, old))
    return {"bytes": keys * hk * d * 2 * 2 + total * hq * d * 2 * 2, "flops": 4 * d * hq * pairs}


# -- inputs --------------------------------------------------------------------------

def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(case, keys, gen, first=0):
    """A table [batch, pages] of pages in no order, for so many keys of each sequence; -1 where there is none."""
    page = case["page"]
    count = torch.tensor([-(-k // page) for k in keys], device="cuda")
    width = max(1, max(-(-k // page) for k in keys))
    total = sum(-(-k // page) for k in keys)
    order = torch.randperm(total, generator=gen, device="cuda") + first
    table = torch.full((len(keys), width), -1, dtype=torch.int64, device="cuda")
    table[torch.arange(width, device="cuda") < count[:, None]] = order
    return table.to(torch.int32), first + total


def _fill(case, pages, tables, gen):
    """Keys and values of the pool; slots that hold no key are NaN, as memory that nothing has written may be."""
    page, dtype = case["page"], DTYPES[case["dtype"]]
    shape = (pages, case["kv_heads"], page, case["head_dim"])
    pool = [torch.randn(shape, generator=gen, device="cuda", dtype=dtype) for _ in range(2)]
    held = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    for table, keys in tables:
        at = torch.arange(table.shape[1] * page, device="cuda")
        slot = table.long()[:, at // page] * page + at % page
        held[slot[at < torch.tensor(keys, device="cuda")[:, None]]] = True
    for t in pool:
        t.masked_fill_(~held.view(pages, 1, page, 1), math.nan)
    return pool


def _rotary(positions, rot):
    """cos and sin [positions, rot / 2] of base 1e6, each angle taken in 64 bits."""
    freq = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, gen)
    new, old = _lengths(case)
    batch, hq, hk, d = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"]
    dtype, total = DTYPES[case["dtype"]], sum(new)
    ends = [0]
    for n in new:
        ends.append(ends[-1] + n)
    state = {"case": case, "new": new, "old": old, "cu": _int32(ends) if case["ragged"] else None,
             "most": max(new), "starts": _int32(ends[:-1]), "count": _int32(new)}
    if case["op"] == "append":
        # The projections' outputs as one tensor, q, k and v beside each other in each token's row.
        qkv = torch.randn(total, hq + 2 * hk, d, generator=gen, device="cuda", dtype=dtype)
        state["q"], state["k"], state["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        state["table"], pages = _pages(case, [n + m for n, m in zip(new, old)], gen)
        shape = (pages, hk, case["page"], d)
        state["k_cache"] = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
        state["v_cache"] = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
        state["cos"], state["sin"] = _rotary(max(n + m for n, m in zip(new, old)), case["rot"])
        state["lengths"] = _int32(old)
        return state
    # Queries of a trained model make scores that differ by more than unit-normal ones do.
    state["q"] = (torch.randn(total, hq, d, generator=gen, device="cuda") * 1.5).to(dtype)
    keys, pages, tables = [n + m for n, m in zip(new, old)], 0, []
    if case["op"] == "prefix":
        table, pages = _pages(case, [case["prefix"]], gen)
        state["prefix_table"], state["prefix"] = table[0].contiguous(), case["prefix"]
        tables.append((table, [case["prefix"]]))
    state["table"], pages = _pages(case, keys, gen, pages)
    tables.append((state["table"], keys))
    state["k_cache"], state["v_cache"] = _fill(case, pages + 3, tables, gen)
    state["lengths"] = _int32(keys)
    return state


def _prepare_verify(case, gen):
    batch, drafts, vocab = case["batch"], case["drafts"], case["vocab"]
    logits = torch.randn(batch, drafts + 1, vocab, generator=gen, device="cuda") * 2.5
    noise = torch.randn(batch, drafts, vocab, generator=gen, device="cuda") * 0.5
    draft = torch.softmax(logits[:, :-1] + noise, dim=-1)
    # A token of each of the draft's distributions: the largest of p / (an exponential number).
    race = -torch.log1p(-torch.rand(batch, drafts, vocab, generator=gen, device="cuda"))
    tokens = (draft / race.clamp_min(1e-30)).argmax(dim=-1)
    return {"case": case, "target": torch.softmax(logits, dim=-1), "draft": draft, "tokens": tokens,
            "uniforms": torch.rand(batch, drafts + 1, generator=gen, device="cuda"),
            "counts": _int32(_drafted(case)) if case["ragged"] else None}


# -- one pass ----------------------------------------------------------------------------

def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


def _own_append(s):
    q = _framework().b200_rope_paged_append(
        s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["cos"], s["sin"],
        cu_tokens=s["cu"], interleaved=s["case"]["interleaved"])
    return q, s["k_cache"], s["v_cache"]


def _own_attention(s):
    return _framework().b200_paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"],
                                             cu_tokens=s["cu"], max_tokens=s["most"])


def _own_prefix(s):
    return _framework().b200_shared_prefix_attention(
        s["q"], s["k_cache"], s["v_cache"], s["prefix_table"], s["prefix"], s["table"], s["lengths"],
        cu_tokens=s["cu"], max_tokens=s["most"])


def _own_verify(s):
    return _framework().b200_verify_draft(s["tokens"], s["target"], s["uniforms"], draft_probs=s["draft"],
                                          draft_counts=s["counts"])


def _owners(s):
    """For each new token its sequence and its place among the sequence's new tokens."""
    t = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted((s["starts"] + s["count"]).long(), t, right=True)
    return b, t - s["starts"].long()[b]


def _turn(x, cos, sin, interleaved):
    """Rotary positions in 32 bits: pairs (i, i + rot / 2), or (2 i, 2 i + 1), of the first rot dimensions."""
    half = cos.shape[-1]
    x = x.float()
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_append(s):
    case, dtype = s["case"], s["q"].dtype
    b, i = _owners(s)
    at = s["lengths"].long()[b] + i
    cos, sin = s["cos"][at], s["sin"][at]
    page = s["table"].long()[b, at // case["page"]]
    s["k_cache"][page, :, at % case["page"]] = _turn(s["k"], cos, sin, case["interleaved"]).to(dtype)
    s["v_cache"][page, :, at % case["page"]] = s["v"]
    return _turn(s["q"], cos, sin, case["interleaved"]).to(dtype), s["k_cache"], s["v_cache"]


def _gather(pool, table):
    """Pages -> [batch, kv_heads, keys, head_dim] in 32 bits."""
    x = pool[table.long().clamp_min(0)].float()
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s, keys, values, seen):
    """Softmax attention in 32 bits: queries padded to [batch, tokens], `seen` [batch, tokens, keys]."""
    q = s["q"]
    hk, group = keys.shape[1], q.shape[1] // keys.shape[1]
    first, most = s["starts"].long(), s["most"]
    slot = (first[:, None] + torch.arange(most, device="cuda")).clamp_max(max(q.shape[0] - 1, 0))
    x = q[slot].float().view(len(first), most, hk, group, -1).permute(0, 2, 3, 1, 4)
    values = values.masked_fill(~seen.any(dim=1)[:, None, :, None], 0)
    score = (x @ keys.transpose(-1, -2)[:, :, None]) * q.shape[-1] ** -0.5
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    weight = torch.exp(score - top.masked_fill(top == -math.inf, 0))
    total = weight.sum(dim=-1, keepdim=True)
    out = (weight @ values[:, :, None]) / total.masked_fill(total == 0, 1)
    b, i = _owners(s)
    return out[b, :, :, i].flatten(1, 2).to(q.dtype)


def _visible(s, width):
    """[batch, tokens, width]: token i of a sequence with n new ones sees its keys up to length - n + i."""
    i = torch.arange(s["most"], device="cuda")
    last = (s["lengths"] - s["count"])[:, None] + i
    last = torch.where(i < s["count"][:, None], last, -1)
    return torch.arange(width, device="cuda") <= last[..., None]


def _plain_attention(s):
    keys, values = _gather(s["k_cache"], s["table"]), _gather(s["v_cache"], s["table"])
    return _attend(s, keys, values, _visible(s, keys.shape[2]))


def _plain_prefix(s):
    batch, table = len(s["new"]), s["prefix_table"][None]
    both = []
    for pool in (s["k_cache"], s["v_cache"]):
        head = _gather(pool, table)[:, :, :s["prefix"]].expand(batch, -1, -1, -1)
        both.append(torch.cat((head, _gather(pool, s["table"])), dim=2))
    seen = _visible(s, both[0].shape[2] - s["prefix"])
    new = torch.arange(s["most"], device="cuda") < s["count"][:, None]
    seen = torch.cat((new[..., None].expand(-1, -1, s["prefix"]), seen), dim=-1)
    return _attend(s, *both, seen)


def _plain_verify(s):
    """Draft i of a sequence stands if u_i q_i(token) < p_i(token) and all before it stand. The token after the a
    that stand is drawn from max(p_a - q_a, 0), or from p_a where no draft was refused, at the row's last uniform
    number (which no draft was tested against): the first v whose running sum of the weights, in units of 2^-40, is
    above that share of their sum."""
    target, draft, tokens, u = s["target"], s["draft"], s["tokens"], s["uniforms"]
    batch, most, vocab = draft.shape
    count = s["counts"].long() if s["counts"] is not None else torch.full((batch,), most, device="cuda")
    place = torch.arange(most, device="cuda")
    p = target[:, :most].gather(-1, tokens[..., None])[..., 0]
    q = draft.gather(-1, tokens[..., None])[..., 0]
    stands = (u[:, :most] * q < p) & (place < count[:, None])
    accepted = stands.long().cumprod(dim=-1).sum(dim=-1)
    b = torch.arange(batch, device="cuda")
    row = target[b, accepted]
    less = draft[b, accepted.clamp_max(max(most - 1, 0))]
    refused = (accepted < count)[:, None]
    weight = torch.where(refused, (row - less).clamp_min(0), row)
    units = (weight.clamp_max(1) * 2.0 ** 40).to(torch.int64)
    whole = (row.clamp(0, 1) * 2.0 ** 40).to(torch.int64)
    units = torch.where(units.sum(dim=-1, keepdim=True) == 0, whole, units)
    running = units.cumsum(dim=-1)
    total = running[:, -1]
    share = (u[:, most] * 2.0 ** 24).to(torch.int64)
    goal = share * (total >> 24) + ((share * (total & (2 ** 24 - 1))) >> 24)
    follows = (running <= goal[:, None]).sum(dim=-1)
    at = torch.arange(most + 1, device="cuda")
    padded = torch.cat((tokens, tokens.new_zeros(batch, 1)), dim=-1)
    out = torch.where(at < accepted[:, None], padded, torch.where(at == accepted[:, None], follows[:, None], -1))
    return out, accepted.to(torch.int32)


# -- the definition in 64 bits -------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "prefix": _exact_attention,
            "verify": _exact_verify}[case["op"]](s)


def _exact_append(s):
    """Each pair of a head's dimensions as one complex number, turned by its position's."""
    case = s["case"]
    n = s["cos"].shape[1]
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    pools = [s["k_cache"].double(), s["v_cache"].double()]
    q, k, v = (s[x].double().clone() for x in "qkv")
    even = slice(0, 2 * n, 2) if case["interleaved"] else slice(0, n)
    odd = slice(1, 2 * n, 2) if case["interleaved"] else slice(n, 2 * n)
    begin = 0
    for b, (new, old) in enumerate(zip(s["new"], s["old"])):
        rows = slice(begin, begin + new)
        for x in (q, k):
            z = torch.complex(x[rows, :, even], x[rows, :, odd]) * turn[old:old + new, None]
            x[rows, :, even], x[rows, :, odd] = z.real, z.imag
        at = torch.arange(old, old + new, device="cuda")
        page = s["table"][b].long()[torch.div(at, case["page"], rounding_mode="floor")]
        for pool, x in zip(pools, (k, v)):
            pool[page, :, at % case["page"]] = x[rows]
        begin += new
    return (q, *pools)


def _exact_attention(s):
    case = s["case"]
    d, hk = case["head_dim"], case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    begin, shared = 0, s.get("prefix", 0)

    def keys_of(pool, table, count, h):
        x = pool[table[:-(-count // case["page"])].long(), h].double()
        return x.reshape(-1, d)[:count]

    for b, (new, old) in enumerate(zip(s["new"], s["old"])):
        for h in range(hk if new else 0):
            k, v = (keys_of(pool, s["table"][b], new + old, h) for pool in (s["k_cache"], s["v_cache"]))
            if shared:
                k = torch.cat((keys_of(s["k_cache"], s["prefix_table"], shared, h), k))
                v = torch.cat((keys_of(s["v_cache"], s["prefix_table"], shared, h), v))
            for i in range(0, new, 512):
                rows = slice(begin + i, begin + min(new, i + 512))
                heads = slice(h * (case["q_heads"] // hk), (h + 1) * (case["q_heads"] // hk))
                x = s["q"][rows, heads].double()
                last = shared + old + i + torch.arange(x.shape[0], device="cuda")
                score = torch.einsum("thd,kd->thk", x, k) / math.sqrt(d)
                hidden = torch.arange(len(k), device="cuda") > last[:, None, None]
                share = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1)
                out[rows, heads] = torch.einsum("thk,kd->thd", share, v)
        begin += new
    return out


def _exact_verify(s):
    """Each sequence by itself, in Python's whole numbers."""
    target, draft = s["target"], s["draft"]
    batch, most, vocab = draft.shape
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    count = s["counts"].tolist() if s["counts"] is not None else [most] * batch
    out, accepted = [], []
    for b in range(batch):
        a = 0
        while a < count[b]:
            t = tokens[b][a]
            product = torch.tensor(u[b][a], dtype=torch.float32) * draft[b, a, t].cpu()
            if not bool(product < target[b, a, t].cpu()):
                break
            a += 1
        p = target[b, a].double()
        w = (p - draft[b, a].double()).float().double().clamp(0, 1) if a < count[b] else p.clamp(0, 1)
        units = torch.floor(w * 2.0 ** 40).long()
        if int(units.sum()) == 0:
            units = torch.floor(p.clamp(0, 1) * 2.0 ** 40).long()
        goal = int(u[b][most] * 2 ** 24) * int(units.sum()) >> 24
        follows = int(torch.searchsorted(units.cumsum(0), goal, right=True))
        out.append(tokens[b][:a] + [follows] + [-1] * (most - a))
        accepted.append(a)
    return torch.tensor(out, device="cuda"), torch.tensor(accepted, dtype=torch.int32, device="cuda")
