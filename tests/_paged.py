"""Plain 64-bit forms of the paged-cache operators, and batches to run them on (no framework code)."""

import math
import random

import torch

# Largest relative rounding error of a value to each type.
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def build(seqs, *, Hq, Hkv, D, page, dtype, device, seed=0, slots_first=False, spare=2, prefix=0, wide=3, scale=1.5):
    """A ragged batch: seqs is [(new tokens, keys in all)]. Pages in random order among `spare` unused ones; every
    slot that holds no key is NaN. With `prefix`, so many shared keys precede every sequence's own."""
    g = torch.Generator(device=device).manual_seed(seed)
    rng = random.Random(seed)
    counts = [-(-max(k, 0) // page) for _, k in seqs]
    npre = -(-prefix // page)
    total = sum(counts) + npre + spare
    order = list(range(total))
    rng.shuffle(order)
    shape = (total, page, Hkv, D) if slots_first else (total, Hkv, page, D)
    kc, vc = (torch.randn(shape, generator=g, device=device).to(dtype) for _ in range(2))
    if slots_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    held = torch.zeros(total, page, dtype=torch.bool)
    width = max(1, max(counts)) + wide
    table = torch.full((len(seqs), width), -1, dtype=torch.int32)
    at = 0

    def take(keys, n):
        nonlocal at
        pages = order[at:at + n]
        at += n
        for j, p in enumerate(pages):
            held[p, :min(page, keys - j * page)] = True
        return pages

    pre = take(prefix, npre)
    for b, ((_, k), n) in enumerate(zip(seqs, counts)):
        table[b, :n] = torch.tensor(take(k, n), dtype=torch.int32)
    dead = ~held.to(device)
    for c in (kc, vc):
        c.masked_fill_(dead[:, None, :, None], math.nan)
    news = [n for n, _ in seqs]
    T = sum(news)
    q = (torch.randn(T, Hq, D, generator=g, device=device) * scale).to(dtype)
    cu = torch.tensor([0] + [sum(news[:i + 1]) for i in range(len(news))], dtype=torch.int32)
    lengths = torch.tensor([k for _, k in seqs], dtype=torch.int32)
    i32 = dict(dtype=torch.int32, device=device)
    return dict(q=q, k=kc, v=vc, table=table.to(device), lengths=lengths.to(device), cu=cu.to(device), seqs=seqs,
                prefix=prefix, prefix_table=torch.tensor(pre, **i32), page=page, most=max(news), Hkv=Hkv, D=D)


def keys_of(pool, pages, count):
    """[Hkv, count, D] in 64 bits."""
    if count <= 0:
        return pool.new_zeros(pool.shape[1], 0, pool.shape[3], dtype=torch.float64)
    x = pool[pages.long()].double()
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :count]


def attention64(batch, *, causal=True, scale=None):
    """(out, out over |V|) [T, Hq, D] in 64 bits."""
    q, page = batch["q"].double(), batch["page"]
    T, Hq, D = q.shape
    Hkv = batch["Hkv"]
    scale = D ** -0.5 if scale is None else scale
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    t0 = 0
    for b, (n, length) in enumerate(batch["seqs"]):
        pages = batch["table"][b, :-(-max(length, 0) // page)]
        k, v = (keys_of(batch[c], pages, length) for c in "kv")
        if batch["prefix"]:
            k, v = (torch.cat((keys_of(batch[c], batch["prefix_table"], batch["prefix"]), x), dim=1)
                    for c, x in (("k", k), ("v", v)))
        for i in range(0, n, 256):
            m = min(256, n - i)
            x = q[t0 + i:t0 + i + m].view(m, Hkv, Hq // Hkv, D)
            s = torch.einsum("thgd,hkd->thgk", x, k) * scale
            sees = length - n + i + torch.arange(m, device=q.device) if causal else torch.full(
                (m,), length - 1, device=q.device)
            sees = sees.clamp_min(-1)  # no own key; a prefix is seen whole
            hidden = torch.arange(k.shape[1], device=q.device) > (sees + batch["prefix"])[:, None]
            s = s.masked_fill(hidden[:, None, None], -math.inf)
            top = s.amax(-1, keepdim=True) if k.shape[1] else s.new_zeros(*s.shape[:-1], 1)
            w = torch.exp(s - top.masked_fill(top == -math.inf, 0))
            w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
            out[t0 + i:t0 + i + m] = torch.einsum("thgk,hkd->thgd", w, v).reshape(m, Hq, D)
            size[t0 + i:t0 + i + m] = torch.einsum("thgk,hkd->thgd", w, v.abs()).reshape(m, Hq, D)
        t0 += n
    return out, size


def check_attention(got, batch, **how):
    """Elementwise bound: the result's own rounding; the weights' rounding to the cache's type at most (u times the
    same weights over |V|); and 2^-13 of that for the FP32 scores (a sum of D products with relative error D 2^-24,
    times scores below 2^4), the exponentials and the sums."""
    ref, size = attention64(batch, **how)
    u = ROUND[got.dtype]
    bound = u * ref.abs() + (u + 2.0 ** -13) * size + 1e-30
    err = (got.double() - ref).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((err <= bound).all()), f"worst {(err / bound).max():.3f} of the bound"


def rotate64(x, cos, sin, interleaved):
    """x [T, heads, D], cos / sin [T, rot / 2], in 64 bits."""
    x = x.double().clone()
    h = cos.shape[-1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    i = slice(0, 2 * h, 2) if interleaved else slice(0, h)
    j = slice(1, 2 * h, 2) if interleaved else slice(h, 2 * h)
    a, b = x[..., i].clone(), x[..., j].clone()
    x[..., i], x[..., j] = a * c - b * s, b * c + a * s
    return x


def verify_plain(tokens, target, uniforms, draft, counts):
    """One sequence at a time, whole numbers in Python."""
    B, K = tokens.shape
    out, accepted = [], []
    target, uniforms, tokens = target.cpu(), uniforms.cpu(), tokens.cpu()
    draft = None if draft is None else draft.cpu()

    def units(w):
        w = w.float()
        w = torch.where(w > 0, w, torch.zeros_like(w)).clamp_max(1.0)  # a NaN counts as nothing
        return torch.floor(w.double() * 2.0 ** 40).long()

    for b in range(B):
        n = K if counts is None else max(0, min(int(counts[b]), K))
        a = 0
        while a < n:
            t = int(tokens[b, a])
            if not 0 <= t < target.shape[2]:
                break
            q = torch.tensor(1.0) if draft is None else draft[b, a, t].float()
            if not bool(uniforms[b, a] * q < target[b, a, t].float()):
                break
            a += 1
        p = target[b, a].float()
        w = p
        if a < n:
            if draft is None:
                w = p.clone()
                if 0 <= int(tokens[b, a]) < len(p):
                    w[int(tokens[b, a])] = 0
            else:
                w = p - draft[b, a].float()
        x = units(w)
        if int(x.sum()) == 0:
            x = units(p)
        total = int(x.sum())
        goal = int(float(uniforms[b, K]) * 2 ** 24) * total >> 24
        follows = int((x.cumsum(0) <= goal).sum()) if total else -1
        out.append(tokens[b, :a].tolist() + [follows] + [-1] * (K - a))
        accepted.append(a)
    return torch.tensor(out, dtype=torch.int64).reshape(B, K + 1), torch.tensor(accepted, dtype=torch.int32)
