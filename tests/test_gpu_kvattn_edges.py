"""The operators over KV caches where their documentation makes a promise that
ordinary inputs do not try: values that are not finite under weights of
nothing, empty batches, captured and threaded calls, blocks that give up."""
import math

import pytest
import torch

from cascade_b200 import kvattn
from test_gpu_kvattn import Case

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def far_apart(heads, cached, low_key, low_score):
    """One token, alike for all heads, whose cached keys score `low_score` or
    100: low in every other tile of 128 keys, the poisoned key's among them.
    The weight of a low key is exp(-200) or less, which is 0 in 32 bits."""
    c = Case([1], [cached], heads, 1, 64, "fp16", seed=90)
    c.q[:] = 0
    c.q[..., 0] = 40.0                        # score = 40 k[0] / 8
    for t in range(cached):
        low = (t // 128) % 2 == (low_key // 128) % 2
        c.pool[c.table[0, t // 16], 0, 0, t % 16, 0] = \
            (low_score if low else 100.0) / 5.0
    c.k[..., 0] = 20.0
    return c


@pytest.mark.parametrize("heads", [2, 32, 256])
@pytest.mark.parametrize("cached", [700, 6000])
@pytest.mark.parametrize("low_score", [-100.0, -math.inf])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("key", [5, 250])
def test_bad_values_show_whatever_their_weight(heads, cached, low_score,
                                               value, key):
    # 0 * inf is NaN: a row that sees a value that is not finite is not
    # finite, whichever part of the kernel the key falls to
    c = far_apart(heads, cached, key, low_score)
    clean, lse = c.run()
    assert clean.isfinite().all()
    c.pool[c.table[0, key // 16], 1, 0, key % 16, ::5] = value
    out, lse2 = c.run()
    assert torch.equal(lse, lse2)
    assert not out[0, :, ::5].isfinite().any()
    rest = torch.arange(64, device=DEV) % 5 != 0
    assert torch.equal(out[0, :, rest], clean[0, :, rest])


@pytest.mark.parametrize("new", [[0], [0, 0, 0]])
def test_weights_of_batches_without_tokens(new):
    plan = kvattn.WeightsPlan(new, q_heads=4, kv_heads=2, head_dim=64,
                              device=DEV)
    q = torch.zeros(0, 4, 64, dtype=torch.float16, device=DEV)
    k = torch.zeros(0, 2, 64, dtype=torch.float16, device=DEV)
    lse = torch.zeros(0, 4, device=DEV)
    assert kvattn.attention_weights(plan, q, k, lse).shape == (len(new), 2, 0)
    # positions behind the sequences are there all the same
    before = torch.rand(len(new), 2, 7, device=DEV)
    got = kvattn.attention_weights(plan, q, k, lse, add_to=before)
    assert torch.equal(got, before)
    out = torch.full_like(before, 3.0)
    kvattn.attention_weights(plan, q, k, lse, add_to=before, out=out)
    assert (out == 3).all()


@pytest.mark.parametrize("heads", [2, 32, 256])
def test_no_pages_at_all(heads):
    # a prefix of which the store held nothing: its tokens count as unseen
    c = Case([3, 1], [300, 40], heads, 1, 64, "bf16", seed=91)
    c.table[:] = 0
    empty = c.pool[:0]
    got, lse = kvattn.prompt_attention(
        c.plan(), c.q, c.k, c.v, (empty[:, 0], empty[:, 1]), c.table)
    c.table[:] = -1
    want = c.run()
    assert torch.equal(got, want[0]) and torch.equal(lse, want[1])
    wplan = c.plan(kvattn.WeightsPlan)
    assert torch.equal(
        kvattn.attention_weights(wplan, c.q, c.k, lse, empty[:, 0], c.table),
        kvattn.attention_weights(wplan, c.q, c.k, lse, c.pages[0], c.table))


@pytest.mark.parametrize("new,heads", [([1, 1, 1], 4), ([90, 3, 40], 4)])
def test_a_page_table_that_the_call_before_writes(new, heads):
    # the heaviest pages of each sequence, chosen on the device into the same
    # tensor as the step before: the attention call may be launched while
    # the choice still runs
    pages, kept = 400, 60
    c = Case(new, [kept * 16] * 3, heads, 2, 64, "bf16", seed=92)
    g = torch.Generator(device=DEV).manual_seed(3)
    c.pool = torch.randn(pages, 2, 2, 16, 64, generator=g,
                         device=DEV).bfloat16()
    scores = torch.rand(6, 3, pages, generator=g, device=DEV)
    plan, wplan = c.plan(), c.plan(kvattn.WeightsPlan)

    def steps(wait):
        outs = []
        for s in scores:
            table = kvattn.select_kept(s, kept)
            wait()
            out, lse = kvattn.prompt_attention(plan, c.q, c.k, c.v, c.pages,
                                               table)
            wait()
            outs += [out, lse, kvattn.attention_weights(
                wplan, c.q, c.k, lse, c.pages[0], table)]
            wait()
            del table             # the next choice is written to its memory
        return outs
    want = steps(torch.cuda.synchronize)
    for _ in range(5):
        assert all(map(torch.equal, steps(lambda: None), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = steps(lambda: None)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(map(torch.equal, got, want))


def test_a_plan_that_the_stream_writes_before_the_call():
    # a caller of the C ABI may keep one device buffer for its plans and
    # fill it by a kernel of the same stream right before the call
    shapes = [([1, 1, 1], [700, 30, 5000]), ([64, 9, 1], [2000, 0, 3]),
              ([300, 2, 17], [100, 9, 1000])]
    cases = [Case(*s, 8, 2, 64, "bf16", seed=93) for s in shapes]
    plans = [(c.plan(), c.plan(kvattn.WeightsPlan)) for c in cases]
    assert any(p._info.merges for ps in plans for p in ps)
    want = []
    for c, (p, w) in zip(cases, plans):
        out, lse = c.run(p)
        want.append((out, lse, kvattn.attention_weights(
            w, c.q, c.k, lse, c.pages[0], c.table)))
    bufs = [[p._buf for p in ps] for ps in plans]
    shared = torch.zeros(max(b.numel() for bs in bufs for b in bs),
                         dtype=torch.int32, device=DEV)
    for ps in plans:
        for p in ps:
            p._ptr = shared.data_ptr()

    def write(b):
        torch.bitwise_or(b, 0, out=shared[:b.numel()])
    for _ in range(10):
        for c, (p, w), (pb, wb), (o0, l0, w0) in zip(cases, plans, bufs,
                                                     want):
            write(pb)
            out, lse = c.run(p)
            write(wb)
            got = kvattn.attention_weights(w, c.q, c.k, lse, c.pages[0],
                                           c.table)
            assert torch.equal(out, o0) and torch.equal(lse, l0)
            assert torch.equal(got, w0)


GIVES_UP = """
import ctypes, itertools, math, sys, torch
sys.path.insert(0, "tests")
from cascade_b200 import _lib, kvattn
from test_gpu_kvattn import Case
give_up = _lib.load().cascade_diag_attn_give_up
give_up.argtypes, give_up.restype = [ctypes.c_int32], None

def calls(c):
    out, lse = c.run()
    return out, lse, None if c.tree else kvattn.attention_weights(
        c.plan(kvattn.WeightsPlan), c.q, c.k, c.run()[1], c.pages[0], c.table)

def same(a, b):
    return all(x is y or torch.equal(x, y) for x, y in zip(a, b))

def run(new, cached, heads, dim, page, tree):
    c = Case(new, cached, heads, 2, dim, "bf16", page=page, tree=tree, seed=94)
    want = calls(c)
    torch.cuda.synchronize()
    for i in range(4):
        before = kvattn.wait_timeouts()
        give_up(1)
        got = calls(c)
        torch.cuda.synchronize()
        assert kvattn.wait_timeouts() > before
        give_up(0)
        assert same(calls(c), want)
        CHECK

for form in (([1], [3000], 4), ([1, 1], [9000, 300], 64), ([130], [900], 4),
             ([300, 20], [0, 4000], 16), ([5] * 90, [30] * 90, 4),
             ([1] * 300, [70] * 300, 8)):
    for dim, page, tree in itertools.product((64, 128), (16, 37), (False, True)):
        run(*form, dim, page, tree)
print("gave up and went on")
"""


def gives_up(check):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", GIVES_UP.replace(
        "CHECK", check)], cwd=root, text=True, capture_output=True,
        timeout=240)
    assert "gave up and went on" in r.stdout, r.stderr[-2000:]


def test_calls_after_one_that_gave_up():
    # in a process of its own, since the others expect no wait to run out
    gives_up("pass")


def test_results_of_calls_that_gave_up_are_nan():
    gives_up("""out, lse, w = got
        assert out.isnan().all() and lse.isnan().all()
        for b, n in enumerate(a + b for a, b in zip(new, cached)):
            assert w is None or w[b, :, :n].isnan().all()
            assert w is None or (w[b, :, n:] == 0).all()
        rows = sum(new)          # nothing else is written
        q, k, v = (torch.cat([t, t[:1]]) for t in (c.q, c.k, c.v))
        o, l = torch.full_like(q, 7.0), torch.full((rows + 1, heads), 7.0,
                                                   device=q.device)
        give_up(1)
        if tree:
            kvattn.tree_attention(c.plan(), q, k, v, torch.cat(
                [c.mask, c.mask[:1]]), c.pages, c.table, out=o, lse=l)
        else:
            kvattn.prompt_attention(c.plan(), q, k, v, c.pages, c.table,
                                    out=o, lse=l)
        give_up(0)
        assert (o[rows:] == 7).all() and (l[rows:] == 7).all()
        assert o[:rows].isnan().all() and l[:rows].isnan().all()""")


@pytest.mark.parametrize("new,cached,heads,kv_heads,page,tree", [
    ([70, 30, 5], [0, 0, 0], 16, 4, 16, False),
    ([1500, 700], [0, 0], 32, 8, 16, False),
    ([400, 90], [9000, 40], 32, 8, 16, False),
    ([1], [1000], 32, 8, 16, True), ([1] * 20, [3000] * 20, 32, 8, 37, True),
    ([64, 64], [4096, 100], 64, 8, 16, True)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_equal_calls_have_equal_results(new, cached, heads, kv_heads, page,
                                        tree, dtype):
    # sums are taken in a fixed order, whatever the blocks' timing
    c = Case(new, cached, heads, kv_heads, 128, dtype, page=page, tree=tree,
             seed=95)
    plan, wplan = c.plan(), c.plan(kvattn.WeightsPlan)

    def calls():
        out, lse = c.run(plan)
        return out, lse, kvattn.attention_weights(
            wplan, c.q, c.k, lse, c.pages[0], c.table)
    want = calls()
    for _ in range(10):
        assert all(map(torch.equal, calls(), want))


def test_every_thread_gets_its_results():
    # errors of a thread are raised by result()
    from concurrent.futures import ThreadPoolExecutor
    cases = [Case([2, 40], [900, 10], 8, 2, 64, "bf16", seed=96 + i)
             for i in range(4)]
    plans = [(c.plan(), c.plan(kvattn.WeightsPlan)) for c in cases]

    def calls(c, plan, wplan):
        out, lse = c.run(plan)
        w = kvattn.attention_weights(wplan, c.q, c.k, lse, c.pages[0],
                                     c.table)
        return out, lse, w, kvattn.select_kept(w, 9, 2, 1)
    want = [calls(c, *p) for c, p in zip(cases, plans)]
    torch.cuda.synchronize()

    def work(i):
        done, s = 0, torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = calls(cases[i], *plans[i])
                s.synchronize()
                done += all(map(torch.equal, got, want[i]))
        return done
    with ThreadPoolExecutor(4) as pool:
        assert [f.result() for f in
                [pool.submit(work, i) for i in range(4)]] == [20] * 4


@pytest.mark.parametrize("width", [8193, 20000, 32768])
def test_select_many_rows_beyond_one_block_of_512(width):
    # more rows than clusters for them: one block of 1024 a row, ties in it
    g = torch.Generator(device=DEV).manual_seed(width)
    w = torch.randn(400, width, generator=g, device=DEV).mul(50).round()
    w[7] = 1.0
    keep = kvattn.select_kept(w, 3001, 100, 4)
    w[:, :4] = math.inf
    w[:, width - 100:] = math.inf
    want = w.sort(dim=1, descending=True, stable=True).indices[
        :, :3001].sort(1).values
    assert torch.equal(keep.long(), want)


@pytest.mark.parametrize("window", [None, 1])
@pytest.mark.parametrize("heads", [2, 64])
def test_weights_of_cached_tokens_alone(window, heads):
    # sequences without new tokens keep what they had
    for new, cached in (([0, 0], [300, 1]), ([0, 3], [1000, 40])):
        c = Case(new, cached, heads, 2, 64, "fp16", seed=97)
        plan = c.plan(kvattn.WeightsPlan, window=window)
        lse = c.run()[1]
        before = torch.rand(2, 2, plan.max_keys + 5, device=DEV)
        got = kvattn.attention_weights(plan, c.q, c.k, lse, c.pages[0],
                                       c.table, add_to=before)
        assert torch.equal(got[0], before[0])
        zero = kvattn.attention_weights(plan, c.q, c.k, lse, c.pages[0],
                                        c.table)
        assert (zero[0] == 0).all()


def test_choices_and_evictions_of_nothing():
    keep = kvattn.select_kept(torch.zeros(3, 2, 0, device=DEV), 4, 1, 1)
    assert keep.shape == (3, 2, 4) and (keep == -1).all()
    assert kvattn.select_kept(torch.zeros(0, 9, device=DEV), 4).shape == (0,
                                                                          4)
    kv = torch.zeros(1, 2, 0, 64, dtype=torch.float16, device=DEV)
    got, keep = kvattn.evict_kv_caches([[(kv, kv)]], torch.zeros(
        1, 2, 0, device=DEV), 5, 2, 1)
    assert got.shape == (1, 1, 2, 2, 0, 64) and keep.shape == (1, 2, 0)
    # no pages: every token of the choice is a row of zeros
    pages = torch.zeros(0, 2, 16, 64, dtype=torch.float16, device=DEV)
    w = torch.rand(3, 2, 40, device=DEV)
    table = torch.zeros(3, 3, dtype=torch.int32, device=DEV)
    lengths = torch.tensor([40, 3, 0], dtype=torch.int32, device=DEV)
    k, v, keep = kvattn.evict_pages(pages, pages, table, lengths, w, 5)
    assert (k == 0).all() and (v == 0).all()
    assert torch.equal((keep >= 0).sum(-1), torch.tensor(
        [[5, 5], [3, 3], [0, 0]], device=DEV))
    k, v, keep = kvattn.evict_pages(pages, pages, table[:0], lengths[:0],
                                    w[:0], 5)
    assert k.shape == (0, 2, 5, 64) and keep.shape == (0, 2, 5)
