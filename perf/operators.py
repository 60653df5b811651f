"""The operators over KV caches (cascade_b200.kvattn), as they are measured.

Four operators that a server runs around the block store, each with its plain
form in elementary torch operations:

* prompt: causal attention of packed prompts with grouped heads, over tokens
  loaded from the store in pages and the prompts' own;
* tree: attention of drafted tokens, each seeing the cached pages and the
  drafts its mask names (one draft is an ordinary decode step);
* weights: the attention weight each cached token received, summed over
  queries and the heads of a group;
* evict: the tokens to keep by that weight, and the shorter cache.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # five short prompts that arrive together: launch latency counts
        dict(name="prompt-short-ragged", op="prompt", dtype="fp16", batch=5,
             new=70, cached=0, heads=16, kv_heads=4, dim=64, page=0),
        # a packed prefill step of ordinary prompts, llama3-8b heads
        dict(name="prompt-packed-8b", op="prompt", dtype="bf16", batch=8,
             new=1500, cached=0, heads=32, kv_heads=8, dim=128, page=0),
        # one long document, llama3-70b heads
        dict(name="prompt-16k-70b", op="prompt", dtype="bf16", batch=1,
             new=16384, cached=0, heads=64, kv_heads=8, dim=128, page=0),
        # questions on prefixes that came from the store as 16-token blocks
        dict(name="prompt-on-stored-prefix", op="prompt", dtype="fp16",
             batch=4, new=400, cached=9000, heads=32, kv_heads=8, dim=128,
             page=16),
        # one user's next token
        dict(name="decode-one", op="tree", dtype="fp16", batch=1, new=1,
             cached=1000, heads=32, kv_heads=8, dim=128, page=16),
        # a batch of users of different history, one token each
        dict(name="decode-batch-64", op="tree", dtype="bf16", batch=64, new=1,
             cached=6000, heads=32, kv_heads=8, dim=128, page=16),
        # drafted trees verified over cached prefixes, llama3-70b heads
        dict(name="tree-64-drafts-70b", op="tree", dtype="bf16", batch=8,
             new=64, cached=4096, heads=64, kv_heads=8, dim=128, page=16),
        # the last 32 queries of prompts weigh the tokens before them
        dict(name="weights-window-32", op="weights", dtype="fp16", batch=4,
             new=2048, cached=0, window=32, heads=32, kv_heads=8, dim=128,
             page=0),
        # each decode step adds its weights, over a batch's cached pages
        dict(name="weights-decode-batch", op="weights", dtype="bf16",
             batch=32, new=1, cached=6000, window=0, heads=32, kv_heads=8,
             dim=128, page=16),
        # a whole prompt's weights
        dict(name="weights-whole-prompt", op="weights", dtype="bf16", batch=1,
             new=8192, cached=0, window=0, heads=32, kv_heads=8, dim=128,
             page=0),
        # a small cache halved before it is stored
        dict(name="evict-small", op="evict", dtype="fp16", batch=1, layers=4,
             kv_heads=8, dim=128, length=300, budget=150, recent=16, sink=4,
             page=0),
        # four llama3-8b caches of 8192 tokens cut to 1024
        dict(name="evict-8b-8k", op="evict", dtype="fp16", batch=4, layers=32,
             kv_heads=8, dim=128, length=8192, budget=1024, recent=64, sink=4,
             page=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "tree", "weights", "evict"])
    kv_heads = rng.choice([1, 2, 4, 8])
    c = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), kv_heads=kv_heads,
             dim=rng.choice([64, 128]))
    if op == "evict":
        c["page"] = rng.choice([0, 0, 16, 24, 64])
        c["length"] = _log(rng, 20, 40000)
        c["batch"] = rng.randint(1, 4)
        c["layers"] = 1 if c["page"] else max(1, min(
            32, _log(rng, 1, 32), 2 ** 28 // (c["length"] * c["batch"] *
                                              kv_heads * c["dim"])))
        c["budget"] = max(2, int(c["length"] * rng.uniform(0.05, 0.9)))
        c["recent"] = rng.randint(0, c["budget"] // 2)
        c["sink"] = rng.randint(0, min(4, c["budget"] - c["recent"]))
        return c
    c["heads"] = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    if op == "tree":
        c["new"] = rng.choice([1, 1, _log(rng, 2, 80)])
        c["cached"] = _log(rng, 1, 30000)
        c["batch"] = max(1, min(_log(rng, 1, 64), 200000 // c["cached"],
                                2 ** 24 // (c["cached"] * c["heads"])))
        c["page"] = rng.choice([8, 16, 16, 37, 64])
        return c
    c["new"] = _log(rng, 3, 6000)
    c["batch"] = max(1, min(_log(rng, 1, 16), 12000 // c["new"]))
    c["page"] = rng.choice([0, 16, 37])
    c["cached"] = _log(rng, 1, 10000) if c["page"] else 0
    if op == "weights":
        c["window"] = rng.choice([0, 16, 33])
    return c


# ----------------------------------------------------------------- inputs
def _spread(mean, batch, seed):
    """`batch` lengths around `mean`, the first one `mean` itself: the ragged
    lengths of a batch.  They depend on the case alone, as work() does."""
    g = torch.Generator().manual_seed(seed)
    f = 0.4 + 0.6 * torch.rand(batch, generator=g)
    out = [max(1, int(mean * float(x))) for x in f]
    out[0] = mean
    return out


def _lengths(case):
    b = case["batch"]
    if case["op"] == "tree":
        new = [case["new"]] * b
    else:
        new = _spread(case["new"], b, 11)
    cached = _spread(case["cached"], b, 12) if case["cached"] else [0] * b
    return new, cached


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _pages(g, lengths, page, kv_heads, dim, dt):
    """Pages in the layout that blocks loaded from the store have for one
    layer ([pages, K and V, heads, page, dim]), and a shuffled page table."""
    counts = [-(-n // page) for n in lengths]
    total, most = sum(counts), max(max(counts), 1)
    pool = torch.empty(max(total, 1), 2, kv_heads, page, dim, dtype=dt,
                       device=DEV)
    step = max(1, 2 ** 27 // (2 * kv_heads * page * dim))
    for s in range(0, pool.shape[0], step):
        p = pool[s:s + step]
        p.copy_(_randn(g, *p.shape))
    ids = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lengths), most), -1, dtype=torch.int32,
                       device=DEV)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    return pool, table


def _tree_mask(g, new):
    """Random trees: each draft hangs on an earlier one or on the context,
    and sees itself and its ancestors."""
    rows = []
    most = max(new)
    for n in new:
        m = torch.zeros(n, most, dtype=torch.bool)
        parent = [-1] + [int(torch.randint(-1, i, (1,), generator=g))
                         for i in range(1, n)]
        for i in range(n):
            if parent[i] >= 0:
                m[i] = m[parent[i]]
            m[i, i] = True
        rows.append(m)
    return torch.cat(rows).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = dict(case=case)
    if case["op"] == "evict":
        return _prepare_evict(case, g, dt, st)
    new, cached = _lengths(case)
    n, H, G, D = sum(new), case["heads"], case["kv_heads"], case["dim"]
    # one projection's output, split by heads, as a model has it
    qkv = _randn(g, n, H + 2 * G, D)
    qkv[:, :H] *= 1.5
    qkv = qkv.to(dt)
    st.update(q=qkv[:, :H], k=qkv[:, H:H + G], v=qkv[:, H + G:], new=new,
              cached=cached, pages=None, table=None)
    if case["page"]:
        pool, st["table"] = _pages(g, cached, case["page"], G, D, dt)
        st["pages"] = (pool[:, 0], pool[:, 1])
    if case["op"] == "tree":
        st["mask"] = _tree_mask(torch.Generator().manual_seed(seed), new)
    if case["op"] == "weights":
        st["window"] = case["window"] or max(new)
        st["lse"] = _plain_attention(st, lse_only=True)
        width = max(a + b for a, b in zip(new, cached))
        before = torch.rand(len(new), G, width, generator=g, device=DEV)
        for b in range(len(new)):
            before[b, :, new[b] + cached[b]:] = 0
        st["before"] = before
    if own:
        from cascade_b200 import kvattn
        more = dict(q_heads=H, kv_heads=G, head_dim=D, device=DEV,
                    page_size=case["page"] or None)
        if case["op"] == "weights":
            st["plan"] = kvattn.WeightsPlan(new, cached, window=st["window"],
                                            **more)
        else:
            st["plan"] = kvattn.AttentionPlan(
                new, cached, tree=case["op"] == "tree", **more)
    return st


def _prepare_evict(case, g, dt, st):
    n, L, G, D = case["batch"], case["layers"], case["kv_heads"], case["dim"]
    S = case["length"]
    lead = (n, G) if case["page"] else (n, L, G)
    # accumulated weights are heavy-tailed, and many tokens got next to none
    w = torch.exp(2.5 * _randn(g, *lead, S)) - 0.3
    st["weights"] = torch.clamp(w, min=0.0)
    if case["page"]:
        st["lengths"] = _spread(S, n, 12)
        st["dev_lengths"] = torch.tensor(st["lengths"], dtype=torch.int32,
                                         device=DEV)
        pool, st["table"] = _pages(g, st["lengths"], case["page"], G, D, dt)
        st["pages"] = (pool[:, 0], pool[:, 1])
        return st
    caches = []
    for _ in range(n):
        kv = [torch.empty(1, G, S, D, dtype=dt, device=DEV)
              for _ in range(2 * L)]
        for t in kv:
            t.copy_(_randn(g, *t.shape))
        caches.append(tuple(zip(kv[0::2], kv[1::2])))
    st["caches"] = caches
    return st


# ------------------------------------------------------------ plain forms
def _sequence(st, b, at):
    """K and V of sequence b, cached tokens then new ones, [kv heads, keys,
    dim] each, in the inputs' type."""
    n, c = st["new"][b], st["cached"][b]
    k, v = (st[x][at:at + n].transpose(0, 1) for x in "kv")
    if c:
        page = st["case"]["page"]
        ids = st["table"][b, :-(-c // page)].long()
        old = [p[ids].transpose(0, 1).flatten(1, 2)[:, :c]
               for p in st["pages"]]
        k, v = torch.cat([old[0], k], 1), torch.cat([old[1], v], 1)
    return k, v


def _visible(st, b, at, i0, i1):
    """[rows, keys]: which keys the new tokens i0..i1 of sequence b see."""
    n, c = st["new"][b], st["cached"][b]
    keys = torch.arange(c + n, device=DEV)
    if "mask" in st:
        m = torch.ones(i1 - i0, c + n, dtype=torch.bool, device=DEV)
        m[:, c:] = st["mask"][at + i0:at + i1, :n]
        return m
    return keys[None, :] <= c + torch.arange(i0, i1, device=DEV)[:, None]


def _blocks(st, rows_of=None):
    """(b, first packed token, i0, i1) over all sequences, in pieces whose
    scores take about a gigabyte."""
    H, at = st["case"]["heads"], 0
    for b, (n, c) in enumerate(zip(st["new"], st["cached"])):
        step = max(1, 2 ** 28 // (H * (n + c)))
        first = 0 if rows_of is None else max(0, n - rows_of)
        for i0 in range(first, n, step):
            yield b, at, i0, min(n, i0 + step)
        at += n


def _scores(st, b, at, i0, i1, k):
    """Scaled scores [kv heads, group, rows, keys] in 32 bits, minus infinity
    where a key is not seen."""
    H, G, D = (st["case"][x] for x in ("heads", "kv_heads", "dim"))
    q = st["q"][at + i0:at + i1].float().view(i1 - i0, G, H // G, D)
    q = q.permute(1, 2, 0, 3).reshape(G, -1, D)
    s = torch.matmul(q, k.transpose(1, 2)).view(G, H // G, i1 - i0, -1)
    s *= 1.0 / math.sqrt(D)
    return s.masked_fill_(~_visible(st, b, at, i0, i1), -math.inf)


def _plain_attention(st, lse_only=False):
    q, case, held = st["q"], st["case"], -1
    out = torch.zeros(q.shape, dtype=q.dtype, device=DEV)
    lse = torch.zeros(q.shape[:2], device=DEV)
    G, D = case["kv_heads"], case["dim"]
    for b, at, i0, i1 in _blocks(st):
        if b != held:
            k, v = (t.float() for t in _sequence(st, b, at))
            held = b
        s = _scores(st, b, at, i0, i1, k)
        top = s.amax(-1, keepdim=True)
        s.sub_(top).exp_()
        total = s.sum(-1, keepdim=True)
        rows = slice(at + i0, at + i1)
        lse[rows] = (top + total.log()).view(-1, i1 - i0).t()
        if not lse_only:
            o = torch.matmul(s.view(G, -1, s.shape[-1]), v).view(
                *s.shape[:3], D) / total
            out[rows] = o.view(-1, i1 - i0, D).transpose(0, 1).to(q.dtype)
    return lse if lse_only else (out, lse)


def _plain_weights(st):
    w, held = st["before"].clone(), -1
    H, G = st["case"]["heads"], st["case"]["kv_heads"]
    for b, at, i0, i1 in _blocks(st, st["window"]):
        if b != held:
            k = _sequence(st, b, at)[0].float()
            held = b
        s = _scores(st, b, at, i0, i1, k)
        lse = st["lse"][at + i0:at + i1].t().view(G, H // G, i1 - i0, 1)
        w[b, :, :s.shape[-1]] += s.sub_(lse).exp_().sum((1, 2))
    return w


def _plain_keep(w, budget, recent, sink):
    """The positions to keep of each row of w [..., length], ascending: the
    first `sink`, the last `recent`, then by weight, ties to the lowest."""
    S = w.shape[-1]
    at = torch.arange(S, device=DEV)
    fixed = (at < sink) | (at >= S - recent)
    order = torch.argsort(w, dim=-1, descending=True, stable=True)
    first = torch.argsort((~fixed[order]).to(torch.uint8), dim=-1, stable=True)
    order = order.gather(-1, first)[..., :budget]
    return order.sort(-1).values


def _plain_evict(st):
    case = st["case"]
    rule = case["recent"], case["sink"]
    w = st["weights"]
    if case["page"]:
        n, G, S = w.shape
        B, D = case["budget"], case["dim"]
        keep = torch.full((n, G, B), -1, dtype=torch.int32, device=DEV)
        kv = [torch.zeros(n, G, B, D, dtype=p.dtype, device=DEV)
              for p in st["pages"]]
        for b, length in enumerate(st["lengths"]):
            m = min(B, length)
            at = _plain_keep(w[b, :, :length], m, *rule)
            keep[b, :, :m] = at
            ids = st["table"][b, :-(-length // case["page"])].long()
            for t, p in zip(kv, st["pages"]):
                rows = p[ids].transpose(0, 1).flatten(1, 2)
                t[b, :, :m] = rows.gather(1, at[..., None].expand(-1, -1, D))
        return kv[0], kv[1], keep
    at = _plain_keep(w, min(case["budget"], w.shape[-1]), *rule)
    kv = torch.stack([torch.stack([torch.stack(
        [t[0].gather(1, at[i, l, :, :, None].expand(-1, -1, t.shape[-1]))
         for t in pair]) for l, pair in enumerate(cache)])
        for i, cache in enumerate(st["caches"])])
    return kv, at.to(torch.int32)


def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return {"prompt": _plain_attention, "tree": _plain_attention,
                "weights": _plain_weights, "evict": _plain_evict}[op](st)
    from cascade_b200 import kvattn
    if op == "prompt":
        return kvattn.prompt_attention(st["plan"], st["q"], st["k"], st["v"],
                                       st["pages"], st["table"])
    if op == "tree":
        return kvattn.tree_attention(st["plan"], st["q"], st["k"], st["v"],
                                     st["mask"], st["pages"], st["table"])
    if op == "weights":
        return kvattn.attention_weights(
            st["plan"], st["q"], st["k"], st["lse"],
            st["pages"][0] if st["pages"] else None, st["table"],
            add_to=st["before"])
    rule = dict(recent=case["recent"], sink=case["sink"])
    if case["page"]:
        return kvattn.evict_pages(*st["pages"], st["table"],
                                  st["dev_lengths"], st["weights"],
                                  case["budget"], **rule)
    return kvattn.evict_kv_caches(st["caches"], st["weights"],
                                  case["budget"], **rule)


# ------------------------------------------------- what a pass cannot avoid
def work(case):
    D, G = case["dim"], case["kv_heads"]
    if case["op"] == "evict":
        n, L = case["batch"], case["layers"]
        lengths = (_spread(case["length"], n, 12) if case["page"]
                   else [case["length"]] * n)
        kept = sum(min(case["budget"], x) for x in lengths)
        per = L * G
        return dict(bytes=per * (4 * sum(lengths) + 4 * kept
                                 + 2 * 2 * 2 * D * kept), flops=0)
    new, cached = _lengths(case)
    H, tokens = case["heads"], sum(new)
    rows = new
    if case["op"] == "tree":
        pairs = sum(n * (c + (n + 1) / 2) for n, c in zip(new, cached))
    else:
        window = case.get("window") or max(new)
        rows = [min(n, window) for n in new]
        pairs = sum(r * (c + n) - r * (r - 1) / 2
                    for r, n, c in zip(rows, new, cached))
    if case["op"] == "weights":
        keys = sum(new) + sum(cached)
        return dict(bytes=2 * D * (G * keys + H * sum(rows))
                    + 4 * (H * sum(rows) + 2 * G * keys),
                    flops=2 * D * H * pairs)
    return dict(bytes=2 * D * (2 * H * tokens + 2 * G * (tokens
                                                         + sum(cached)))
                + 4 * H * tokens, flops=4 * D * H * pairs)


# ------------------------------------------------------------- in 64 bits
def _exact_heads(st):
    """For each sequence and query head: packed rows, scores [new, keys] and
    V in 64 bits, from the definition."""
    case, at = st["case"], 0
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    for b, (n, c) in enumerate(zip(st["new"], st["cached"])):
        for h in range(H):
            kv = h // (H // G)
            parts = []
            for x, p in (("k", 0), ("v", 1)):
                t = st[x][at:at + n, kv].double()
                if c:
                    tok = torch.arange(c, device=DEV)
                    ids = st["table"][b].long()[tok // case["page"]]
                    t = torch.cat([st["pages"][p][ids, kv, tok % case["page"]]
                                   .double(), t])
                parts.append(t)
            for i0 in range(0, n, 8192):
                i1 = min(n, i0 + 8192)
                s = st["q"][at + i0:at + i1, h].double() @ parts[0].t()
                s /= math.sqrt(D)
                late = torch.zeros_like(s, dtype=torch.bool)
                if "mask" in st:
                    late[:, c:] = ~st["mask"][at + i0:at + i1, :n]
                else:
                    late = torch.ones_like(late).triu(c + 1 + i0)
                s[late] = -math.inf
                yield b, h, at + i0, i0, s, parts[1]
        at += n


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(st)
    if case["op"] == "weights":
        w = st["before"].double()
        for b, h, at, i0, s, _ in _exact_heads(st):
            skip = max(0, st["new"][b] - st["window"] - i0)
            if skip < s.shape[0]:
                rows = st["lse"][at + skip:at + s.shape[0], h].double()
                p = torch.exp(s[skip:] - rows[:, None])
                kv = h * case["kv_heads"] // case["heads"]
                w[b, kv, :s.shape[1]] += p.sum(0)
        return w
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(st["q"].shape[:2], dtype=torch.float64, device=DEV)
    for b, h, at, i0, s, v in _exact_heads(st):
        rows = slice(at, at + s.shape[0])
        lse[rows, h] = torch.logsumexp(s, 1)
        out[rows, h] = torch.exp(s - lse[rows, h, None]) @ v
    return out, lse


def _exact_evict(st):
    """By the threshold: what is above the last kept weight, and the lowest
    positions among those equal to it."""
    case, w = st["case"], st["weights"].double()
    n, G, D = case["batch"], case["kv_heads"], case["dim"]
    paged = bool(case["page"])
    lengths = st["lengths"] if paged else [case["length"]] * n
    B = case["budget"] if paged else min(case["budget"], case["length"])
    w = w if not paged else w[:, None]
    keep = torch.full((*w.shape[:3], B), -1, dtype=torch.int64, device=DEV)
    kv = torch.zeros((n, w.shape[1], 2, G, B, D), dtype=torch.float64,
                     device=DEV)
    for b, S in enumerate(lengths):
        m = min(B, S)
        x = w[b, :, :, :S].clone()
        x[..., :case["sink"]] = math.inf
        x[..., max(0, S - case["recent"]):] = math.inf
        least = x.sort(-1, descending=True).values[..., m - 1:m]
        equal = x == least
        room = m - (x > least).sum(-1, keepdim=True)
        kept = (x > least) | (equal & (equal.cumsum(-1) <= room))
        at = kept.nonzero()[:, -1].view(*x.shape[:2], m)
        keep[b, :, :, :m] = at
        head = torch.arange(G, device=DEV)[:, None]
        for l in range(w.shape[1]):
            for p in range(2):
                if paged:
                    ids = st["table"][b].long()[at[l] // case["page"]]
                    t = st["pages"][p][ids, head, at[l] % case["page"]]
                else:
                    t = st["caches"][b][l][p][0][head, at[l]]
                kv[b, l, p, :, :m] = t.double()
    if paged:
        return kv[:, 0, 0], kv[:, 0, 1], keep[:, 0]
    return kv, keep
