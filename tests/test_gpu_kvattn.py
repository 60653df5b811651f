"""The attention operators over KV caches (cascade_b200.kvattn) against plain
formulas in 64 bits.

Tolerances, from the roundings that the kernels make (u = eps / 2 of the
16-bit type): the output is rounded once (u |o|), the softmax weights are
rounded to the type before they multiply V (u A, A = sum p |v|), scores and
sums are in FP32.  A score's error is at most d = dim 2^-23 max_j scale sum
|q k|, which moves a weight by a factor of up to exp(2 d); sums over n keys
add n 2^-23 at most, and the exponential 2^-21."""
import math

import pytest
import torch

from cascade_b200 import kvattn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def paged(gen, lengths, page, heads, dim, dt, cols=None, spare=2):
    """Random pages (K and V interleaved as a loaded block has them), a
    shuffled table, and each sequence's (k, v) [heads, tokens, dim]."""
    counts = [-(-n // page) for n in lengths]
    P = sum(counts) + spare
    pool = torch.randn(P, 2, heads, page, dim, generator=gen,
                       device=DEV).to(dt)
    ids = torch.randperm(P, generator=gen, device=DEV).to(torch.int32)
    cols = max(counts + [1]) if cols is None else cols
    table = torch.full((len(lengths), cols), -1, dtype=torch.int32,
                       device=DEV)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = ids[at:at + c]
        at += c
    return pool, table


def cached_rows(pool, table, b, n, page):
    tok = torch.arange(n, device=DEV)
    ids = table[b].long()[tok // page] if n else tok
    ok = (ids >= 0) & (ids < pool.shape[0])
    rows = pool[ids.clamp(0, pool.shape[0] - 1), :, :, tok % page]
    return rows[:, 0], rows[:, 1], ok      # [n, heads, dim]


class Case:
    def __init__(self, new, cached, heads, kv_heads, dim, dtype, page=16,
                 tree=False, seed=0, scale=None, mask=None, qmul=1.5):
        g = torch.Generator(device=DEV).manual_seed(seed + 1)
        self.new, self.cached, self.page = new, cached, page
        self.H, self.G, self.D, self.dt = heads, kv_heads, dim, DT[dtype]
        n = sum(new)
        qkv = torch.randn(n, heads + 2 * kv_heads, dim, generator=g,
                          device=DEV)
        qkv[:, :heads] *= qmul
        qkv = qkv.to(self.dt)
        self.q = qkv[:, :heads]
        self.k = qkv[:, heads:heads + kv_heads]
        self.v = qkv[:, heads + kv_heads:]
        self.pool, self.table = paged(g, cached, page, kv_heads, dim,
                                      self.dt)
        self.tree, self.scale = tree, scale
        if tree and mask is None:
            m = torch.rand(n, max(new), generator=g, device=DEV) < 0.5
            at = 0
            for c in new:
                i = torch.arange(c, device=DEV)
                m[at + i, i] = True
                at += c
            mask = m
        self.mask = mask

    def plan(self, cls=kvattn.AttentionPlan, **kw):
        if cls is kvattn.AttentionPlan:
            kw["tree"] = self.tree
        return cls(self.new, self.cached, q_heads=self.H, kv_heads=self.G,
                   head_dim=self.D, page_size=self.page, device=DEV, **kw)

    @property
    def pages(self):
        return self.pool[:, 0], self.pool[:, 1]

    def run(self, plan=None, **kw):
        plan = plan or self.plan()
        if self.tree:
            return kvattn.tree_attention(plan, self.q, self.k, self.v,
                                         self.mask, self.pages, self.table,
                                         scale=self.scale, **kw)
        return kvattn.prompt_attention(plan, self.q, self.k, self.v,
                                       self.pages, self.table,
                                       scale=self.scale, **kw)

    def sequences(self):
        """(b, first token, keys k, v [heads, keys, dim], visible [new,
        keys]) in 64 bits."""
        at = 0
        for b, (n, c) in enumerate(zip(self.new, self.cached)):
            ck, cv, ok = cached_rows(self.pool, self.table, b, c, self.page)
            k = torch.cat([ck, self.k[at:at + n]]).double().transpose(0, 1)
            v = torch.cat([cv, self.v[at:at + n]]).double().transpose(0, 1)
            vis = torch.zeros(n, c + n, dtype=torch.bool, device=DEV)
            vis[:, :c] = ok
            if self.tree:
                vis[:, c:] = self.mask[at:at + n, :n].bool()
            else:
                i = torch.arange(n, device=DEV)
                vis[:, c:] = i[None, :] <= i[:, None]
            yield b, at, k, v, vis
            at += n

    def scores(self, at, n, k, vis):
        s = self.scale or 1 / math.sqrt(self.D)
        q = self.q[at:at + n].double().transpose(0, 1)
        kk = k.repeat_interleave(self.H // self.G, 0)
        sc = s * q @ kk.transpose(1, 2)
        size = s * q.abs() @ torch.nan_to_num(kk, 0, 0, 0).abs().transpose(
            1, 2)
        d = self.D * 2.0 ** -23 * size.amax(-1) if size.shape[-1] else \
            size.sum(-1)
        return sc.masked_fill(~vis, -math.inf), d


def check_forward(case, out, lse):
    u = torch.finfo(case.dt).eps / 2
    for b, at, k, v, vis in case.sequences():
        n = case.new[b]
        if n == 0:
            continue
        s, d = case.scores(at, n, k, vis)
        want_lse = torch.logsumexp(s, -1)                  # [H, n]
        empty = ~vis.any(-1)
        p = torch.softmax(s, -1).masked_fill(empty[:, None], 0.0)
        vv = v.repeat_interleave(case.H // case.G, 0)
        o, mag = p @ vv, p @ vv.abs()
        slack = 2 * d + s.shape[-1] * 2.0 ** -23 + 2.0 ** -20
        got = out[at:at + n].double().transpose(0, 1)
        tol = u * o.abs() + (u + slack[..., None]) * mag * (1 + 2 * u) + 1e-30
        tol = tol + torch.finfo(case.dt).smallest_normal * u * 2 + \
            (6e-8 if case.dt is torch.float16 else 0)
        bad = (got - o).abs() > tol
        assert not bad.any(), (b, bad.nonzero()[:5].tolist(),
                               float(((got - o).abs() / tol).max()))
        gl = lse[at:at + n].double().t()
        assert (gl[:, empty] == -math.inf).all()
        assert (got[:, empty] == 0).all()
        tl = d + s.shape[-1] * 2.0 ** -23 + 2.0 ** -20 + \
            want_lse.abs() * 2.0 ** -21
        diff = (gl - want_lse)[:, ~empty].abs()
        assert (diff <= tl[:, ~empty]).all(), (b, float(diff.max()))


SHAPES = [
    # new, cached, heads, kv heads, dim, page
    ([1], [0], 4, 1, 64, 16),
    ([1], [1], 8, 8, 128, 1),
    ([5, 0, 1, 130], [0, 9, 0, 0], 4, 2, 64, 16),
    ([1, 1, 1], [127, 128, 129], 32, 8, 128, 16),
    ([33, 7], [300, 64], 7, 1, 128, 37),
    ([128, 64, 129], [0, 1, 255], 2, 2, 64, 8),
    ([300], [77], 8, 2, 128, 16),
    ([1000, 17], [0, 500], 4, 4, 128, 64),
    ([600, 1], [1500, 3], 16, 2, 64, 24),
    ([1], [20000], 8, 1, 128, 16),
    ([2, 1], [9000, 4000], 12, 4, 64, 37),
]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_forward(shape, dtype, tree):
    new, cached, H, G, D, page = SHAPES[shape]
    c = Case(new, cached, H, G, D, dtype, page, tree, seed=shape)
    check_forward(c, *c.run())
    assert kvattn.wait_timeouts() == 0


FORMS = [  # rows: up to 16, up to 128, more; each with parts and merges too
    ([1, 1, 1], 4, 1), ([2, 1], 16, 2), ([3], 5, 1),
    ([9, 4], 4, 1), ([16, 1], 8, 1), ([64, 20], 2, 1),
    ([65, 300], 2, 1), ([40, 129], 8, 2)]


@pytest.mark.parametrize("page", [8, 16, 32, 96, 128, 512])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_forms_and_page_sizes(form, dim, page):
    # page sizes that whole tiles are fetched in, some pages gone, and pages
    # laid out [page, token, head, dim]
    new, H, G = FORMS[form]
    cached = [1300, 127, 5000][:len(new)]
    c = Case(new, cached, H, G, dim, "bf16", page, form % 2 == 1,
             seed=form + page)
    c.table[0, c.table.shape[1] // 3] = -1
    check_forward(c, *c.run())
    other = c.pool.transpose(2, 3).contiguous().transpose(2, 3)
    assert other.stride() != c.pool.stride() or page == 1 or G == 1
    before = c.run()
    c.pool = other
    after = c.run()
    assert torch.equal(before[0], after[0])
    assert torch.equal(before[1], after[1])
    assert kvattn.wait_timeouts() == 0


@pytest.mark.parametrize("scale", [0.01, 0.5])
def test_scale(scale):
    c = Case([40, 3], [200, 90], 4, 2, 128, "fp16", scale=scale, seed=3)
    check_forward(c, *c.run())


def test_large_scores_keep_their_weight():
    # scores far beyond exp's range: the running maximum has to move
    c = Case([50, 1], [500, 700], 4, 2, 64, "bf16", seed=4, qmul=1.0)
    c.q = c.q * 100
    check_forward(c, *c.run())
    c = Case([70], [300], 4, 1, 128, "fp16", seed=5)
    # scores that rise along the keys: the maximum grows in every tile
    ramp = torch.arange(300, device=DEV).view(-1, 1) / 8
    c.q = c.q.clone()
    c.q[:] = 1.0
    ids = c.table[0].long()[torch.arange(300, device=DEV) // 16]
    c.pool[ids, 0, 0, torch.arange(300, device=DEV) % 16] = ramp.to(c.dt)
    check_forward(c, *c.run())


@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (64, 1)])
def test_rows_without_any_key(heads, kv_heads):
    # no cached token and an all-false mask row: zeros and -inf
    new = [6, 40, 3]
    mask = torch.zeros(sum(new), 40, dtype=torch.bool, device=DEV)
    mask[6:46] = torch.rand(40, 40, device=DEV) < 0.2
    mask[10] = False
    c = Case(new, [0, 0, 5], heads, kv_heads, 64, "bf16", tree=True,
             mask=mask, seed=6)
    out, lse = c.run()
    assert (lse[:6] == -math.inf).all() and (out[:6] == 0).all()
    assert (lse[46:] > -math.inf).all()
    check_forward(c, out, lse)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("heads", [2, 16])
def test_pages_that_are_gone_count_as_unseen(tree, heads):
    c = Case([3, 20, 1], [500, 300, 64], heads, 2, 128, "fp16", tree=tree,
             seed=7)
    c.table[0, 3:9] = -1
    c.table[1, 0] = -5
    c.table[1, 7] = c.pool.shape[0]            # behind the last page
    c.table[2] = 2 ** 31 - 1
    check_forward(c, *c.run())


def _poison(c, b, toks, value, which):
    """Writes value into K or V of new tokens of sequence b."""
    at = sum(c.new[:b])
    t = (c.k, c.v)[which]
    for i in toks:
        t[at + i, :, ::3] = value


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("heads", [2, 8, 32])
def test_masked_infinities_do_not_leak(value, which, heads):
    # token 9 of a prompt holds inf or NaN: earlier rows do not see it, later
    # ones do
    c = Case([30, 12], [40, 0], heads, 2, 64, "bf16", seed=8)
    clean, clean_lse = c.run()
    _poison(c, 0, [9, 20], value, which)
    out, lse = c.run()
    assert torch.equal(out[:9], clean[:9])
    assert torch.equal(lse[:9], clean_lse[:9])
    assert torch.equal(out[30:], clean[30:])
    if which == 1:
        assert torch.equal(lse, clean_lse)
        got = out[9:30, :, ::3].float()
        if math.isnan(value):
            assert got.isnan().all()
        else:
            assert (got == value).all()
        rest = torch.ones(64, dtype=torch.bool, device=DEV)
        rest[::3] = False
        assert torch.equal(out[..., rest], clean[..., rest])


def test_masked_infinities_of_a_tree():
    c = Case([8, 70], [20, 300], 8, 2, 128, "fp16", tree=True, seed=9)
    c.mask[:, 5] = False
    c.mask[3, 5] = True
    clean, clean_lse = c.run()
    _poison(c, 0, [5], math.inf, 1)
    _poison(c, 1, [5], math.nan, 1)
    out, lse = c.run()
    seen = c.mask[:, 5]
    assert torch.equal(out[~seen], clean[~seen])
    assert torch.equal(lse, clean_lse)
    assert (out[3, :, ::3] == math.inf).all()


@pytest.mark.parametrize("heads", [2, 32, 128])
@pytest.mark.parametrize("cached", [40, 3000])
def test_all_scores_minus_infinity_is_nan(heads, cached):
    # keys are seen, but no score is above -inf: 0 / 0, not an empty row
    c = Case([2], [cached], heads, 1, 64, "bf16", seed=10)
    c.q = torch.full_like(c.q, 1.0)
    c.k = torch.full_like(c.k, -math.inf)
    c.pool[:, 0] = -math.inf
    out, lse = c.run()
    assert out.isnan().all()


@pytest.mark.parametrize("heads", [2, 32, 256])
def test_scores_of_minus_infinity_weigh_nothing(heads):
    c = Case([1], [600], heads, 1, 64, "bf16", seed=10)
    c.q = torch.full_like(c.q, 1.0)
    clean = c.run()
    ids = c.table[0].long()
    c.pool[ids[:20], 0] = -math.inf
    c2 = c.run()
    c.table[0, :20] = -1
    want = c.run()
    assert torch.equal(c2[0], want[0]) and torch.equal(c2[1], want[1])
    assert not torch.equal(clean[0], want[0])


@pytest.mark.parametrize("heads,new", [(2, 1), (64, 1), (8, 64), (8, 300)])
@pytest.mark.parametrize("cached", [400, 9000])
@pytest.mark.parametrize("sign", [1, -1])
def test_means_of_the_largest_values_stay_finite(heads, new, cached, sign):
    # Every value is the largest of FP16 and 31 of 32 weights round up by
    # nearly half a step, 2^-11: the sum of the products would round to
    # infinity, the mean of such values is that value.
    c = Case([new], [cached], heads, 2, 64, "fp16", seed=11, scale=1.0)
    top = torch.finfo(torch.float16).max
    # p = (1 + 1.1 * 2^-11) / 2, its score as a sum of two halves
    x = math.log(0.5 * (1 + 1.1 * 2.0 ** -11))
    coarse = torch.tensor(x).half()
    fine = torch.tensor(x - float(coarse)).half()
    c.q, c.k, c.v = c.q.clone(), c.k.clone(), c.v.clone()
    c.q.zero_()
    c.q[..., :2] = 1.0
    c.pool[:, 0] = 0.0
    c.pool[:, 0, ..., 0], c.pool[:, 0, ..., 1] = coarse, fine
    c.pool[c.table[0, ::2].long(), 0, :, 0] = 0.0  # p = 1, each 32nd token
    c.pool[:, 1] = sign * top
    c.k.zero_()
    c.k[..., 0], c.k[..., 1] = coarse, fine
    c.v.fill_(sign * top)
    out, lse = c.run()
    # P's roundings 2^-11, the output's 2^-11, sums of n values n 2^-24
    low = top * (1 - 2.0 ** -10 - (cached + new) * 2.0 ** -23)
    assert (out.float() * sign >= low).all() and out.isfinite().all()


@pytest.mark.parametrize("heads,new", [(2, 1), (64, 1), (8, 64), (8, 300)])
@pytest.mark.parametrize("cached", [400, 9000])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_small_weights_beside_a_large_one_of_no_value(heads, new, cached,
                                                      dtype):
    # Each 32nd token takes nearly all weight and has the value 0; the others
    # weigh 11.6 * 2^-24, which has four bits as an FP16 number.
    c = Case([new], [cached], heads, 2, 64, dtype, seed=12, scale=1.0)
    x = math.log(11.6 * 2.0 ** -24)
    coarse = torch.tensor(x).to(c.dt)
    fine = torch.tensor(x - float(coarse)).to(c.dt)
    c.q, c.k, c.v = c.q.clone(), c.k.clone(), c.v.clone()
    c.q.zero_()
    c.q[..., :2] = 1.0
    c.k.zero_()
    c.k[..., 0], c.k[..., 1] = coarse, fine
    c.v.fill_(1000.0)
    c.pool[:, 0] = 0.0
    c.pool[:, 0, ..., 0], c.pool[:, 0, ..., 1] = coarse, fine
    c.pool[:, 1] = 1000.0
    ids = c.table[0, ::2].long()
    c.pool[ids, :, :, 0] = 0.0
    out, lse = c.run()
    check_forward(c, out, lse)


def test_layouts_and_untouched_rows():
    # q, out and lse as slices of larger tensors, K and V as a permuted
    # [heads, tokens, dim] cache, more packed rows than the plan has
    c = Case([40, 9], [100, 33], 8, 2, 64, "fp16", seed=11)
    want, want_lse = c.run()
    n, extra = 49, 7
    big = torch.zeros(n + extra, 3, 8, 64, dtype=c.dt, device=DEV)
    big[:n, 1] = c.q
    kk = torch.zeros(2, n + extra, 80, dtype=c.dt, device=DEV)
    vv = torch.zeros_like(kk)
    kk[:, :n, 8:72] = c.k.transpose(0, 1)
    vv[:, :n, 16:80] = c.v.transpose(0, 1)
    out = torch.full((8, n + extra, 72), 7.0, dtype=c.dt, device=DEV)
    lse = torch.full((8, n + extra), 7.0, device=DEV)
    o, l = kvattn.prompt_attention(
        c.plan(), big[:, 1], kk[:, :, 8:72].transpose(0, 1),
        vv[:, :, 16:80].transpose(0, 1), c.pages, c.table,
        out=out[:, :, :64].transpose(0, 1), lse=lse.t())
    assert o.data_ptr() == out.data_ptr()
    assert torch.equal(o[:n], want) and torch.equal(l[:n], want_lse)
    assert (out[:, n:] == 7).all() and (out[:, :, 64:] == 7).all()
    assert (lse[:, n:] == 7).all()


@pytest.mark.parametrize("heads", [2, 32, 256])
def test_infinities_in_cached_values_stay_with_their_rows(heads):
    c = Case([1, 1], [700, 300], heads, 1, 64, "fp16", seed=16)
    clean = c.run()
    page = int(c.table[0, 20])
    c.pool[page, 1, 0, 3, ::5] = math.inf
    out, lse = c.run()
    assert torch.equal(lse, clean[1]) and torch.equal(out[1], clean[0][1])
    assert not out[0, :, ::5].isfinite().any()
    rest = torch.arange(64, device=DEV) % 5 != 0
    assert torch.equal(out[0, :, rest], clean[0][0, :, rest])


def test_one_vector_for_all_tokens():
    # K and V expanded along the tokens (stride 0): no tensor map for those
    c = Case([300], [0], 4, 2, 64, "bf16", seed=17)
    c.k = c.k[:1].expand(300, 2, 64)
    c.v = c.v[:1].expand(300, 2, 64)
    check_forward(c, *c.run())


def test_contiguous_cache_as_one_page_each():
    # a [sequences, heads, capacity, dim] static cache is a page a sequence
    c = Case([1, 1, 1], [0, 70, 200], 8, 2, 128, "bf16", page=256, seed=12)
    c.table[:] = torch.tensor([[2], [0], [1]], dtype=torch.int32)
    check_forward(c, *c.run())


def test_same_result_twice_and_on_other_streams_and_graphs():
    c = Case([1] * 5, [3000, 10, 700, 5000, 129], 32, 8, 128, "bf16", seed=13)
    plan = c.plan()
    assert plan._info.merges > 0
    want, want_lse = c.run(plan)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(c.run(plan))
    torch.cuda.synchronize()
    for o, l in got:
        assert torch.equal(o, want) and torch.equal(l, want_lse)
    graphs, outs = [], []
    for s in streams[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(c.run(plan))
        graphs.append(g)
    for o, l in outs:
        o.zero_()
    for s, g in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    for o, l in outs:
        assert torch.equal(o, want) and torch.equal(l, want_lse)


def test_offsets_beyond_32_bits():
    # a pool whose last pages start more than 2^32 bytes in
    heads, page, dim = 8, 64, 128
    P = (1 << 32) // (2 * heads * page * dim * 2) + 40
    pool = torch.zeros(P, 2, heads, page, dim, dtype=torch.bfloat16,
                       device=DEV)
    c = Case([1, 2], [600, 300], 16, heads, dim, "bf16", page=page, seed=14)
    ids = torch.randperm(30, device=DEV)[:c.pool.shape[0]] + (P - 31)
    pool[ids] = c.pool
    c.pool = pool
    c.table = torch.where(c.table >= 0, ids[c.table.clamp(min=0).long()]
                          .to(torch.int32), c.table)
    check_forward(c, *c.run())


def test_empty_batches():
    for new, cached in (([], []), ([0, 0], [5, 0])):
        plan = kvattn.AttentionPlan(new, cached, q_heads=4, kv_heads=2,
                                    head_dim=64, page_size=16, device=DEV)
        q = torch.zeros(0, 4, 64, dtype=torch.float16, device=DEV)
        k = torch.zeros(0, 2, 64, dtype=torch.float16, device=DEV)
        pages = (torch.zeros(1, 2, 16, 64, dtype=torch.float16,
                             device=DEV),) * 2
        table = torch.zeros(len(new), 1, dtype=torch.int32, device=DEV)
        out, lse = kvattn.prompt_attention(plan, q, k, k, pages, table)
        assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_refusals():
    c = Case([4, 2], [30, 5], 4, 2, 64, "fp16", seed=15)
    plan, tplan = c.plan(), kvattn.AttentionPlan(
        c.new, c.cached, q_heads=4, kv_heads=2, head_dim=64, page_size=16,
        tree=True, device=DEV)
    mask = torch.ones(6, 4, dtype=torch.bool, device=DEV)

    def call(plan=plan, q=c.q, k=c.k, v=c.v, pages=c.pages, table=c.table,
             **kw):
        return kvattn.prompt_attention(plan, q, k, v, pages, table, **kw)
    call()
    for bad in (dict(q=c.q.float()), dict(q=c.q[:5]), dict(k=c.k[:, :1]),
                dict(q=c.q[..., :32]), dict(k=c.k.bfloat16()),
                dict(q=c.q.cpu()), dict(plan=tplan), dict(pages=None),
                dict(table=None), dict(table=c.table.long()),
                dict(table=c.table[:1]), dict(table=c.table[:, :1]),
                dict(table=c.table.cpu()), dict(pages=(c.pages[0], None)),
                dict(pages=(c.pages[0], c.pages[1][:, :, :8])),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
                dict(scale=math.inf), dict(scale=1e-30), dict(scale=1e30),
                dict(out=torch.empty(6, 4, 64, device=DEV)),
                dict(out=torch.empty(1, 4, 64, dtype=c.dt, device=DEV)
                     .expand(6, 4, 64)),
                dict(lse=torch.empty(6, 4, dtype=torch.float64, device=DEV)),
                dict(plan=c.plan(kvattn.WeightsPlan))):
        with pytest.raises((ValueError, TypeError)):
            call(**bad)
    flat = torch.zeros(6 * 4 * 64 + 1, dtype=c.dt, device=DEV)
    with pytest.raises(ValueError, match="16-byte"):
        call(q=flat[1:].view(6, 4, 64))
    with pytest.raises(RuntimeError, match="backward"):
        call(q=c.q.clone().requires_grad_())
    with torch.no_grad():
        call(q=c.q.clone().requires_grad_())
    for bad in (None, mask[:5], mask[:, :3], mask.float(), mask.cpu()):
        with pytest.raises(ValueError):
            kvattn.tree_attention(tplan, c.q, c.k, c.v, bad, c.pages, c.table)
    with pytest.raises(ValueError):
        kvattn.tree_attention(plan, c.q, c.k, c.v, mask, c.pages, c.table)
    for kw in (dict(new_lengths=[1.5]), dict(new_lengths=[[1]]),
               dict(new_lengths=[1], cached_lengths=[1, 2]),
               dict(new_lengths=[-1]), dict(device="cpu")):
        a = dict(new_lengths=[1], q_heads=4, kv_heads=2, head_dim=64,
                 page_size=16, device=DEV)
        a.update(kw)
        with pytest.raises((ValueError, TypeError)):
            kvattn.AttentionPlan(a.pop("new_lengths"),
                                 a.pop("cached_lengths", None), **a)


# ----------------------------------------------------------------- weights
def check_weights(case, lse, window, got, before):
    for b, at, k, v, vis in case.sequences():
        n, keys = case.new[b], case.new[b] + case.cached[b]
        base = before[b, :, :keys].double() if before is not None else \
            torch.zeros(case.G, keys, dtype=torch.float64, device=DEV)
        g = got[b, :, :keys].double()
        if n == 0:
            assert torch.equal(g, base)
            continue
        s, d = case.scores(at, n, k, vis)
        ll = lse[at:at + n].double().t()
        first = max(0, n - window)
        p = torch.exp(s - ll[..., None])[:, first:]
        p = p.nan_to_num(0.0) if (ll == -math.inf).any() else p
        # a weight's exponent: the score's error, and that of the 32-bit
        # subtraction of lse (both scaled by log2 e and back: 4 roundings)
        rel = d[:, first:, None] + 2.0 ** -22 * (
            4 + 2 * ll[:, first:, None].abs() + s[:, first:].abs()
            .nan_to_num(0, posinf=0))
        w = p.reshape(case.G, -1, keys).sum(1)
        tol = (p * rel).reshape(case.G, -1, keys).sum(1)
        rows = p.shape[1] * case.H // case.G
        # sums: 128 rows by themselves, then the chunks and the parts
        tol = tol + w * 2.0 ** -24 * (128 + rows / 128 + 8) + \
            base.abs() * 2.0 ** -24
        want = base + w
        want = torch.where(vis[first:].any(0) if n else vis, want, base)
        bad = (g - want).abs() > tol + 1e-12
        assert not bad.any(), (b, bad.nonzero()[:5].tolist(),
                               float((g - want).abs().max()))


@pytest.mark.parametrize("window", [None, 1, 33])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_weights(shape, dtype, window):
    new, cached, H, G, D, page = SHAPES[shape]
    c = Case(new, cached, H, G, D, dtype, page, seed=shape + 50)
    out, lse = c.run()
    width = max(a + b for a, b in zip(new, cached)) + 3
    before = torch.rand(len(new), G, width, device=DEV)
    plan = c.plan(kvattn.WeightsPlan, window=window)
    w = kvattn.attention_weights(plan, c.q, c.k, lse, c.pages[0], c.table,
                                 add_to=before)
    check_weights(c, lse, window or 10 ** 9, w, before)
    for b, (n, m) in enumerate(zip(new, cached)):
        assert torch.equal(w[b, :, n + m:], before[b, :, n + m:])
    # each query's weights sum to 1 over the keys it sees
    if window is None:
        w0 = kvattn.attention_weights(plan, c.q, c.k, lse, c.pages[0],
                                      c.table)
        assert w0.shape[2] == width - 3
        check_weights(c, lse, 10 ** 9, w0, None)
        for b, n in enumerate(new):
            assert abs(float(w0[b].double().sum()) - n * H) < 1e-3 * n * H \
                + 1e-6
            assert (w0[b, :, n + cached[b]:] == 0).all()
    assert kvattn.wait_timeouts() == 0


def test_weights_in_place_leaves_the_rest():
    c = Case([3, 1], [300, 20], 8, 2, 128, "fp16", seed=60)
    out, lse = c.run()
    plan = c.plan(kvattn.WeightsPlan)
    args = (plan, c.q, c.k, lse, c.pages[0], c.table)
    big = torch.rand(2, 4, 400, device=DEV)
    acc = big[:, 1:3, 5:320]
    keep = big.clone()
    want = kvattn.attention_weights(*args, add_to=acc)
    got = kvattn.attention_weights(*args, add_to=acc, out=acc)
    assert got.data_ptr() == acc.data_ptr()
    for b, n in enumerate([303, 21]):
        assert torch.equal(acc[b, :, :n], want[b, :, :n])
        assert torch.equal(acc[b, :, n:], keep[b, 1:3, 5 + n:320])
    big[:, 1:3, 5:320] = keep[:, 1:3, 5:320]
    assert torch.equal(big, keep)


def test_weights_of_gone_pages_and_captured():
    c = Case([40, 2], [200, 600], 4, 2, 64, "bf16", seed=61)
    c.table[1, 2:5] = -1
    c.table[0, 0] = c.pool.shape[0] + 3
    out, lse = c.run()
    plan = c.plan(kvattn.WeightsPlan, window=20)
    before = torch.rand(2, 2, 700, device=DEV)
    w = kvattn.attention_weights(plan, c.q, c.k, lse, c.pages[0], c.table,
                                 add_to=before)
    check_weights(c, lse, 20, w, before)
    assert torch.equal(w[1, :, 32:80], before[1, :, 32:80])
    assert torch.equal(w[0, :, :16], before[0, :, :16])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w2 = kvattn.attention_weights(plan, c.q, c.k, lse, c.pages[0],
                                      c.table, add_to=before)
    w2.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(w, w2)


@pytest.mark.parametrize("heads", [2, 8, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_weights_of_keys_that_a_broken_row_does_not_see(value, heads):
    # tokens 9 and 150 of a prompt ask with inf or NaN, so their lse is NaN:
    # the keys behind them were not seen by them
    c = Case([200, 12], [40, 0], heads, 2, 64, "bf16", seed=63)
    plan = c.plan(kvattn.WeightsPlan)

    def weigh(q, lse, plan=plan):
        return kvattn.attention_weights(plan, q, c.k, lse, c.pages[0],
                                        c.table)
    out, lse = c.run()
    clean = weigh(c.q, lse)
    for token, after in ((9, c.plan(kvattn.WeightsPlan)),
                         (150, c.plan(kvattn.WeightsPlan, window=60))):
        q = c.q.clone()
        q[token, :, ::5] = value
        bad = lse.clone()
        bad[token] = math.nan
        want = weigh(c.q, lse, after)
        got = weigh(q, bad, after)
        assert got[0, :, :40 + token + 1].isnan().all()
        assert torch.equal(got[0, :, 40 + token + 1:],
                           want[0, :, 40 + token + 1:])
        assert torch.equal(got[1], want[1])
    assert not clean.isnan().any()


def test_weights_refusals():
    c = Case([4, 2], [30, 5], 4, 2, 64, "fp16", seed=62)
    out, lse = c.run()
    plan = c.plan(kvattn.WeightsPlan)
    w = torch.zeros(2, 2, 34, device=DEV)

    def call(plan=plan, lse=lse, kp=c.pages[0], **kw):
        return kvattn.attention_weights(plan, c.q, c.k, lse, kp, c.table,
                                        **kw)
    call(add_to=w)
    for bad in (dict(plan=c.plan()), dict(lse=lse.double()),
                dict(lse=lse[:5]), dict(kp=None), dict(add_to=w[:, :, :33]),
                dict(add_to=w.double()), dict(out=w[:1]),
                dict(out=torch.zeros(1, 2, 34, device=DEV).expand(2, 2, 34)),
                dict(out=w.transpose(1, 2)), dict(scale=0.0)):
        with pytest.raises((ValueError, TypeError)):
            call(**bad)
    with pytest.raises(ValueError):
        c.plan(kvattn.WeightsPlan, window=0)


# ------------------------------------------------------ calls of all sorts
def test_many_short_sequences():
    n = 3001
    c = Case([1] * n, [(i * 7) % 40 for i in range(n)], 4, 2, 64, "fp16",
             seed=70)
    out, lse = c.run()
    tok = torch.arange(40, device=DEV)
    rows = c.pool[c.table.long()[:, tok // 16].clamp(min=0), :, :, tok % 16]
    k = torch.cat([rows[:, :, 0], c.k[:, None]], 1).double()
    v = torch.cat([rows[:, :, 1], c.v[:, None]], 1).double()
    see = torch.ones(n, 41, dtype=torch.bool, device=DEV)
    see[:, :40] = tok[None] < torch.tensor(c.cached, device=DEV)[:, None]
    s = torch.einsum("nghd,nkgd->nghk", c.q.double().view(n, 2, 2, 64), k) / 8
    s = s.masked_fill(~see[:, None, None], -math.inf)
    want = torch.einsum("nghk,nkgd->nghd", s.softmax(-1), v).view(n, 4, 64)
    # |v| <= 5.5, the weights and the output are rounded once
    assert (out.double() - want).abs().max() < 2 * 2.0 ** -11 * 5.5
    assert (lse.double() - torch.logsumexp(s, -1).view(n, 4)).abs().max() \
        < 1e-4
    w = kvattn.attention_weights(c.plan(kvattn.WeightsPlan), c.q, c.k, lse,
                                 c.pages[0], c.table)
    assert (w.sum(-1) - 2).abs().max() < 1e-3


def test_one_table_row_for_all_sequences():
    # sequences that share a prefix: an expanded table row
    c = Case([3, 1, 2], [200, 200, 200], 8, 2, 128, "bf16", seed=71)
    c.table = c.table[:1].expand(3, -1)
    check_forward(c, *c.run())


def test_mask_of_bytes_and_wider_rows():
    c = Case([5, 9], [30, 4], 4, 2, 64, "fp16", tree=True, seed=72)
    want = c.run()
    wide = torch.zeros(14, 40, dtype=torch.uint8, device=DEV)
    wide[:, 3:12] = c.mask[:, :9].to(torch.uint8) * 7
    c.mask = wide[:, 3:20]
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_from_several_threads():
    import threading
    cases = [Case([2, 40], [900, 10], 8, 2, 64, "bf16", seed=80 + i)
             for i in range(4)]
    want = [c.run() for c in cases]
    plans = [c.plan() for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                out, lse = cases[i].run(plans[i])
                s.synchronize()
                if not torch.equal(out, want[i][0]):
                    bad.append(i)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_first_call_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys
    code = """
import torch
from cascade_b200 import kvattn
plans = [(n, kvattn.AttentionPlan([n], [3000], q_heads=4, kv_heads=1,
                                  head_dim=64, page_size=16))
         for n in (1, 20, 200)]
w = kvattn.WeightsPlan([200], [3000], q_heads=4, kv_heads=1, head_dim=64,
                       page_size=16)
t = torch.arange(188, dtype=torch.int32, device="cuda")[None]
kv = torch.randn(188, 2, 1, 16, 64, device="cuda").half()
ins = [[torch.randn(n, h, 64, device="cuda").half() for h in (4, 1, 1)]
       for n, _ in plans]
def calls():
    r = [kvattn.prompt_attention(p, *x, (kv[:, 0], kv[:, 1]), t)
         for (_, p), x in zip(plans, ins)]
    weights = kvattn.attention_weights(w, ins[2][0], ins[2][1], r[2][1],
                                       kv[:, 0], t)
    keep = kvattn.evict_pages(kv[:, 0], kv[:, 1], t, torch.full(
        (1,), 3000, dtype=torch.int32, device="cuda"), weights, 100)
    return [o for o, _ in r] + [weights, *keep]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = calls()
g.replay()
torch.cuda.synchronize()
a = [x.clone() for x in a]
b = calls()
assert all(torch.equal(x, y) for x, y in zip(a, b))
print("captured first")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, text=True,
                       capture_output=True, timeout=120)
    assert "captured first" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("new,cached,heads", [
    ([1, 1, 1], [700, 30, 5000], 8), ([64, 9], [2000, 0], 16),
    ([900, 300], [0, 100], 4)])
def test_calls_that_feed_each_other_without_a_wait(new, cached, heads):
    # launches may start before the one in front has ended: each call reads
    # what the one before it wrote, into the same buffers, with no other
    # kernel between
    c = Case(new, cached, heads, 2, 64, "bf16", seed=64)
    plan, wplan = c.plan(), c.plan(kvattn.WeightsPlan)
    a, b = c.q.contiguous().clone(), torch.empty_like(c.q.contiguous())
    lse = torch.empty(sum(new), heads, device=DEV)
    acc = torch.zeros(len(new), 2, wplan.max_keys, device=DEV)

    def steps(wait):
        for x, y in ((a, b), (b, a)) * 4:
            kvattn.prompt_attention(plan, x, c.k, c.v, c.pages, c.table,
                                    out=y, lse=lse)
            wait()
            kvattn.attention_weights(wplan, x, c.k, lse, c.pages[0], c.table,
                                     add_to=acc, out=acc)
            wait()
            keep = kvattn.select_kept(acc, 3)
            wait()
        return [t.clone() for t in (a, b, lse, acc, keep)]

    def reset():
        a.copy_(c.q)
        b.zero_()
        acc.zero_()
    reset()
    want = steps(torch.cuda.synchronize)
    for _ in range(5):
        reset()
        assert all(map(torch.equal, steps(lambda: None), want))
    reset()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = steps(lambda: None)
    for _ in range(3):
        reset()
        g.replay()
        torch.cuda.synchronize()
        assert all(map(torch.equal, got, want))
