"""Eviction from KV caches (cascade_b200.kvattn.select_kept, evict_kv_caches,
evict_pages) against sorted references.  Positions and copied rows are exact;
nothing is rounded."""
import math

import numpy as np
import pytest
import torch

from cascade_b200 import cascade_cpp as cc
from cascade_b200 import kvattn, kvwire

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def plain_keep(w, budget, recent, sink):
    """One row, on the host: sort by (fixed, weight, -position)."""
    S = len(w)
    m = min(S, budget)
    if S <= budget:
        return list(range(S))
    fixed = set(range(sink)) | set(range(S - recent, S))
    rank = [-math.inf if math.isnan(x) else x for x in w]
    rest = sorted((i for i in range(S) if i not in fixed),
                  key=lambda i: (-rank[i], i))
    return sorted(fixed | set(rest[:m - len(fixed)]))


def check_keep(w, keep, budget, recent, sink, lengths=None):
    lead = w.shape[:-1]
    w, k = w.cpu().numpy(), keep.cpu().numpy()
    for i in np.ndindex(*lead):
        n = w.shape[-1] if lengths is None else \
            min(max(lengths[i[0]], 0), w.shape[-1])
        want = plain_keep(w[i][:n].tolist(), budget, recent, sink)
        want += [-1] * (budget - len(want))
        assert k[i].tolist() == want, (i, n)


def weights(kind, shape, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.randn(shape, generator=g, device=DEV)
    if kind == "ties":
        return torch.round(w)
    if kind == "heavy":
        return torch.clamp(torch.exp(3 * w) - 0.5, min=0)
    if kind == "equal":
        return torch.full_like(w, 0.25)
    if kind == "odd":
        u = torch.rand(shape, generator=g, device=DEV)
        w[u < 0.1] = math.nan
        w[(u > 0.1) & (u < 0.2)] = -math.inf
        w[(u > 0.2) & (u < 0.3)] = math.inf
        w[(u > 0.3) & (u < 0.4)] = 0.0
        w[(u > 0.4) & (u < 0.5)] = -0.0
        w[(u > 0.5) & (u < 0.6)] = 1e-42
    return w


@pytest.mark.parametrize("kind", ["normal", "ties", "heavy", "equal", "odd"])
@pytest.mark.parametrize("shape,budget,recent,sink", [
    ((1, 1), 1, 0, 0), ((3, 2), 1, 0, 0), ((2, 33), 32, 0, 0),
    ((2, 3, 100), 40, 7, 3), ((4, 1000), 999, 0, 0), ((2, 1000), 5, 3, 2),
    ((2, 2, 2, 777), 300, 16, 4), ((1, 5000), 2500, 100, 4),
    ((3, 20000), 1024, 64, 0), ((2, 517), 600, 20, 4),
    ((1, 65), 64, 0, 64), ((1, 65), 64, 64, 0)])
def test_select(kind, shape, budget, recent, sink):
    w = weights(kind, shape, budget + len(shape))
    keep = kvattn.select_kept(w, budget, recent, sink)
    assert keep.dtype == torch.int32 and keep.shape == (*shape[:-1], budget)
    check_keep(w, keep, budget, recent, sink)


def test_select_long_rows():
    # one row over a whole cluster, and slices beyond shared memory
    for n, rows in ((131072, 1), (400001, 1), (70000, 200)):
        w = weights("heavy", (rows, n), 5)
        keep = kvattn.select_kept(w, n // 3, 10, 4)
        w[:, :4] = math.inf
        w[:, n - 10:] = math.inf
        want = w.sort(dim=1, descending=True, stable=True).indices[
            :, :n // 3].sort(1).values
        assert torch.equal(keep.long(), want)


def test_select_lengths_and_strides():
    big = weights("heavy", (5, 4, 3, 900), 9)
    w = big[:, 1:3, :, 17:817]
    lengths = [0, 1, 800, 10 ** 6, -3]
    dev = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    keep = kvattn.select_kept(w, 90, 8, 2, lengths=dev)
    check_keep(w.contiguous(), keep, 90, 8, 2, lengths)


def test_select_refusals():
    w = torch.rand(2, 10, device=DEV)
    for kw in (dict(budget=0), dict(budget=3, recent=2, sink=2),
               dict(budget=3, recent=-1), dict(budget=3, sink=-1),
               dict(budget=3, lengths=torch.tensor([1, 2], device=DEV)),
               dict(budget=3, lengths=torch.tensor(
                   [1], dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            kvattn.select_kept(w, **kw)
    for bad in (w.cpu(), w.double(), w[0], w.t(), w.view(1, 1, 1, 2, 10)):
        with pytest.raises(ValueError):
            kvattn.select_kept(bad, 3)


def caches(n, L, H, S, D, dt, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def one():
        if dt.is_floating_point:
            return torch.randn(1, H, S, D, generator=g, device=DEV).to(dt)
        return torch.randint(-100, 100, (1, H, S, D), generator=g,
                             device=DEV).to(dt)
    return [tuple((one(), one()) for _ in range(L)) for _ in range(n)]


def check_kv(src, kv, keep):
    for i, cache in enumerate(src):
        for l, pair in enumerate(cache):
            at = (keep[i, l] if keep.dim() == 4 else keep[i]).long()
            for p, t in enumerate(pair):
                want = t.reshape(t.shape[-3:]).gather(
                    1, at[..., None].expand(-1, -1, t.shape[-1]))
                assert torch.equal(kv[i, l, p].view(torch.int16),
                                   want.view(torch.int16))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16,
                                torch.float32])
@pytest.mark.parametrize("n,L,H,S,D,budget", [
    (1, 1, 1, 1, 1, 1), (2, 3, 2, 37, 24, 10), (1, 2, 8, 300, 128, 150),
    (3, 1, 1, 50, 7, 49), (1, 4, 2, 2000, 64, 33), (2, 2, 3, 20, 128, 64),
    (5, 80, 2, 16, 64, 5), (600, 1, 1, 9, 8, 4)])
def test_evict_caches(dt, n, L, H, S, D, budget):
    src = caches(n, L, H, S, D, dt, S)
    for shape in ((n, L, H, S), (n, H, S)):
        w = weights("heavy", shape, budget)
        kv, keep = kvattn.evict_kv_caches(src, w, budget,
                                          min(4, budget // 3),
                                          min(2, budget // 3))
        m = min(budget, S)
        assert kv.shape == (n, L, 2, H, m, D) and kv.dtype == dt
        assert keep.shape == (*shape[:-1], m)
        if S <= 300:
            check_keep(w, keep, m, min(4, budget // 3, m),
                       min(2, budget // 3) if budget < S else 0)
        check_kv(src, kv, keep)


def test_evict_strided_and_unaligned_caches():
    big = torch.randn(2, 2, 3, 60, 40, device=DEV).half()
    sliced = tuple((big[l, 0, :, 5:45, :32], big[l, 1, :, 5:45, :32])
                   for l in range(2))
    perm = torch.randn(2, 2, 40, 3, 32, device=DEV).half()
    permuted = tuple((perm[l, 0].permute(1, 0, 2).unsqueeze(0),
                      perm[l, 1].permute(1, 0, 2).unsqueeze(0))
                     for l in range(2))
    flat = torch.randn(4 * 3 * 40 * 32 + 1, device=DEV).half()[1:]
    odd = tuple((flat[2 * l * 3840:(2 * l + 1) * 3840].view(3, 40, 32),
                 flat[(2 * l + 1) * 3840:(2 * l + 2) * 3840].view(3, 40, 32))
                for l in range(2))
    w = weights("normal", (1, 2, 3, 40), 1)
    for c in (sliced, permuted, odd):
        kv, keep = kvattn.evict_kv_caches([c], w, 11, 2, 1)
        check_kv([c], kv, keep)


@pytest.mark.parametrize("page,D", [(1, 64), (16, 128), (37, 24), (64, 128)])
def test_evict_pages(page, D):
    H, lengths = 3, [0, 1, 200, 333, 40]
    counts = [-(-n // page) for n in lengths]
    g = torch.Generator(device=DEV).manual_seed(page)
    pool = torch.randn(sum(counts) + 3, 2, H, page, D, generator=g,
                       device=DEV).half()
    ids = torch.randperm(pool.shape[0], generator=g, device=DEV).int()
    table = torch.full((5, max(counts) + 1), -1, dtype=torch.int32,
                       device=DEV)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = ids[at:at + c]
        at += c
    w = weights("heavy", (5, H, 350), page)
    dev = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    k, v, keep = kvattn.evict_pages(pool[:, 0], pool[:, 1], table, dev, w,
                                    50, 5, 2)
    check_keep(w, keep, 50, 5, 2, lengths)
    for b in range(5):
        for h in range(H):
            for j, pos in enumerate(keep[b, h].tolist()):
                if pos < 0:
                    assert (k[b, h, j] == 0).all() and (v[b, h, j] == 0).all()
                    continue
                row = pool[int(table[b, pos // page]), :, h, pos % page]
                assert torch.equal(k[b, h, j], row[0])
                assert torch.equal(v[b, h, j], row[1])
                if j > 60:
                    break


def test_evict_pages_that_are_gone():
    # a table entry that names no page, and lengths beyond the table
    pool = torch.ones(4, 2, 2, 8, 64, device=DEV).half()
    table = torch.tensor([[0, -1], [9, 3]], dtype=torch.int32, device=DEV)
    w = torch.rand(2, 2, 30, device=DEV)
    dev = torch.tensor([16, 30], dtype=torch.int32, device=DEV)
    k, v, keep = kvattn.evict_pages(pool[:, 0], pool[:, 1], table, dev, w, 30)
    assert (k[0, :, :8] == 1).all() and (k[0, :, 8:] == 0).all()
    assert (k[1, :, :8] == 0).all() and (k[1, :, 8:16] == 1).all()
    assert (v[1, :, 16:] == 0).all()


def test_evict_refusals():
    src = caches(2, 2, 2, 30, 64, torch.float16, 0)
    w = torch.rand(2, 2, 2, 30, device=DEV)
    other = caches(1, 2, 2, 31, 64, torch.float16, 0)
    for c, ww, kw in (([], w, {}), (src, w[:1], {}), (src, w[..., :29], {}),
                      (src, w.cpu(), {}), (src[:1] + other, w, {}),
                      (src, w, dict(recent=9, sink=2)), (src, w.double(), {}),
                      (src[:1] + caches(1, 1, 2, 30, 64, torch.float16, 0),
                       w, {}),
                      (src[:1] + caches(1, 2, 2, 30, 64, torch.float32, 0),
                       w, {})):
        with pytest.raises(ValueError):
            kvattn.evict_kv_caches(c, ww, 10, **kw)
    kp = torch.zeros(3, 2, 16, 64, device=DEV).half()
    t = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    w = torch.rand(2, 2, 30, device=DEV)
    kvattn.evict_pages(kp, kp, t, n, w, 4)
    for a in ((kp.cpu(), kp, t, n, w), (kp, kp[:2], t, n, w),
              (kp, kp, t.long(), n, w), (kp, kp, t[:1], n, w),
              (kp, kp, t, n.long(), w), (kp, kp, t, n, w[:, :1])):
        with pytest.raises(ValueError):
            kvattn.evict_pages(*a, 4)


def test_evict_refuses_what_needs_a_gradient():
    src = caches(2, 2, 2, 30, 64, torch.float16, 0)
    w = torch.rand(2, 2, 2, 30, device=DEV)
    grad = [[(k.clone().requires_grad_(), v) for k, v in c] for c in src]
    kp = torch.zeros(3, 2, 16, 64, device=DEV).half()
    t = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    n = torch.full((2,), 20, dtype=torch.int32, device=DEV)
    pw = torch.rand(2, 2, 30, device=DEV)
    for f in (lambda: kvattn.evict_kv_caches(grad, w, 10),
              lambda: kvattn.evict_kv_caches(src, w.clone().requires_grad_(),
                                             10),
              lambda: kvattn.select_kept(w.clone().requires_grad_(), 10),
              lambda: kvattn.evict_pages(kp.clone().requires_grad_(), kp, t,
                                         n, pw, 4),
              lambda: kvattn.evict_pages(kp, kp.clone().requires_grad_(), t,
                                         n, pw, 4)):
        with pytest.raises(RuntimeError, match="backward"):
            f()
        with torch.no_grad():
            f()
    # what is stored has no gradient to lose
    store = _store()
    st = kvwire.store_kv_caches(store, ["a", "b"], grad, weights=w, budget=10)
    assert (np.asarray(st) == 0).all()
    got = kvwire.load_kv_caches(store, ["a", "b"], 2, 2, 10, 64)
    kv, _ = kvattn.evict_kv_caches(src, w, 10)
    for i, cache in enumerate(got):
        for l, (k, v) in enumerate(cache):
            assert torch.equal(k[0], kv[i, l, 0])
            assert torch.equal(v[0], kv[i, l, 1])
    store.close()


# ------------------------------------------------------- a run of them all
def _store(gib=1):
    cfg = cc.CascadeConfig()
    cfg.gpu_capacity_bytes = gib << 30
    cfg.shm_capacity_bytes = 64 << 20
    return cc.CascadeStore(cfg)


def test_store_attend_weigh_evict_store_attend():
    """A prefix in the store as 16-token blocks: load its pages, run a
    prompt's rest and a draft tree over them, weigh the tokens, evict, store
    the shorter cache, and attend over that."""
    L, G, H, D, page = 2, 4, 16, 128, 16
    n_blocks, tail = 12, 5                      # cached 11 * 16 + 5 tokens
    cached = (n_blocks - 1) * page + tail
    store = _store()
    blocks = [tuple((torch.randn(1, G, page, D, device=DEV).half(),
                     torch.randn(1, G, page, D, device=DEV).half())
                    for _ in range(L)) for _ in range(n_blocks)]
    ids = [f"prefix-{i}" for i in range(n_blocks)]
    assert (np.asarray(kvwire.store_kv_caches(store, ids, blocks)) == 0).all()
    order = [int(i) for i in torch.randperm(n_blocks)]
    pages, found = kvwire.load_kv_pages(store, [ids[i] for i in order], L, G,
                                        page, D)
    assert found.all() and pages.shape == (n_blocks, L, 2, G, page, D)
    table = torch.tensor([[order.index(i) for i in range(n_blocks)]],
                         dtype=torch.int32, device=DEV)
    missing, found = kvwire.load_kv_pages(store, ["no"], L, G, page, D)
    assert not found.any()
    new = 9
    kw = dict(q_heads=H, kv_heads=G, head_dim=D, page_size=page, device=DEV)
    plan = kvattn.AttentionPlan([new], [cached], **kw)
    wplan = kvattn.WeightsPlan([new], [cached], window=4, **kw)
    full, w_all = [], []
    for l in range(L):
        q, k, v = (torch.randn(new, h, D, device=DEV).half()
                   for h in (H, G, G))
        kv = pages[:, l, 0], pages[:, l, 1]
        out, lse = kvattn.prompt_attention(plan, q, k, v, kv, table)
        w = kvattn.attention_weights(wplan, q, k, lse, kv[0], table)
        # the plain forms over the blocks that were stored
        kk = torch.cat([b[l][0][0] for b in blocks], 1)[:, :cached]
        vv = torch.cat([b[l][1][0] for b in blocks], 1)[:, :cached]
        kk = torch.cat([kk, k.transpose(0, 1)], 1).double()
        vv = torch.cat([vv, v.transpose(0, 1)], 1).double()
        s = q.double().transpose(0, 1) @ kk.repeat_interleave(
            H // G, 0).transpose(1, 2) / math.sqrt(D)
        s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(
            cached + 1), -math.inf)
        p = s.softmax(-1)
        ref = (p @ vv.repeat_interleave(H // G, 0)).transpose(0, 1)
        # |v| <= 5.5; the weights and the output are rounded to fp16 once
        assert (out.double() - ref).abs().max() < 2 * 2.0 ** -11 * 5.5
        # a score is off by 128 2^-23 * 10 at most, a sum of weights is <= 16
        wref = p[:, -4:].reshape(G, -1, cached + new).sum(1)
        assert (w[0].double() - wref).abs().max() < 16 * 1.6e-4
        full.append((kk[:, :cached].half(), vv[:, :cached].half()))
        w_all.append(w[0, :, :cached])
    # evict from the assembled cache while storing it
    cache = tuple((k[None], v[None]) for k, v in full)
    weights = torch.stack(w_all)[None]
    budget = 64
    st = kvwire.store_kv_caches(store, ["short"], [cache], weights=weights,
                                budget=budget, recent=8, sink=2)
    assert (np.asarray(st) == 0).all()
    short = kvwire.load_kv_caches(store, ["short"], L, G, budget, D)[0]
    kv, keep = kvattn.evict_kv_caches([cache], weights, budget, 8, 2)
    assert (keep[..., :2] == torch.arange(2, device=DEV)).all()
    for l in range(L):
        assert torch.equal(short[l][0][0], kv[0, l, 0])
        assert torch.equal(short[l][1][0], kv[0, l, 1])
    # one page of the same layer, evicted in place of the gathered cache
    k1, v1, keep1 = kvattn.evict_pages(
        pages[:, 0, 0], pages[:, 0, 1], table,
        torch.tensor([cached], dtype=torch.int32, device=DEV),
        weights[:, 0].contiguous(), budget, 8, 2)
    assert torch.equal(keep1, keep[:, 0]) and torch.equal(k1[0], kv[0, 0, 0])
    # drafts over the short cache: it is one page of `budget` tokens
    mask = torch.eye(3, dtype=torch.bool, device=DEV)
    tplan = kvattn.AttentionPlan([3], [budget], q_heads=H, kv_heads=G,
                                 head_dim=D, page_size=budget, tree=True,
                                 device=DEV)
    q, k, v = (torch.randn(3, h, D, device=DEV).half() for h in (H, G, G))
    one = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    out, _ = kvattn.tree_attention(tplan, q, k, v, mask,
                                   (short[0][0], short[0][1]), one)
    for i in range(3):
        kk = torch.cat([short[0][0][0], k[i][:, None]], 1).double()
        vv = torch.cat([short[0][1][0], v[i][:, None]], 1).double()
        s = (q[i].double().view(G, H // G, D) @ kk.transpose(1, 2)) \
            / math.sqrt(D)
        ref = (s.softmax(-1) @ vv).view(H, D)
        assert (out[i].double() - ref).abs().max() < 2 * 2.0 ** -11 * 5.5
    with pytest.raises(ValueError):
        kvwire.store_kv_caches(store, ["x"], [cache], weights=weights)
    store.close()


def test_evict_captured_and_on_another_stream():
    src = caches(2, 3, 2, 500, 64, torch.bfloat16, 1)
    w = weights("heavy", (2, 3, 2, 500), 2)
    want, keep = kvattn.evict_kv_caches(src, w, 77, 5, 3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kv, k = kvattn.evict_kv_caches(src, w, 77, 5, 3)
    s.synchronize()
    assert torch.equal(kv, want) and torch.equal(k, keep)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv, k = kvattn.evict_kv_caches(src, w, 77, 5, 3)
    kv.zero_()
    w.mul_(-1.0)                       # other weights, the same graph
    g.replay()
    torch.cuda.synchronize()
    assert not torch.equal(k, keep)
    check_keep(w, k, 77, 5, 3)
    check_kv(src, kv, k)
