"""Plans of the attention operators on a machine without a GPU: every unit of
work of every item is in exactly one segment, parts and merges agree, and
what cannot be planned is refused."""
import ctypes
import random

import numpy as np
import pytest
import torch

from cascade_b200 import _lib, kvattn

TILE = 128


def make(kind, new, cached, heads=32, kv_heads=8, dim=128, page=16, tree=0,
         window=2 ** 31 - 1, sms=148, capacity=None):
    info = kvattn._PlanInfo(kind=kind, batch=len(new), q_heads=heads,
                            kv_heads=kv_heads, head_dim=dim, page_size=page,
                            tree=tree, window=window, sms=sms)
    n, c = np.array(new, np.int32), np.array(cached, np.int32)
    for size in ([1 << 12, None] if capacity is None else [capacity]):
        buf = np.full(size or info.ints, -7, np.int32)
        rc = _lib.load().cascade_attn_plan(
            ctypes.byref(info), n.ctypes.data, c.ctypes.data,
            buf.ctypes.data, buf.size)
        _lib.check(rc)
        if info.ints <= buf.size:
            break
    return info, buf


def split(info, buf):
    first = buf[:info.ctas + 1]
    at = -(-(info.ctas + 1) // 16) * 16
    segs = buf[at:at + 16 * info.segments].reshape(-1, 16)
    at += 16 * info.segments
    return first, segs, buf[at:at + 8 * info.merges].reshape(-1, 8)


def units(kind, new, cached, group, kv_heads, row_tile, tree, window):
    """{(b, head, row0, key0): (range of units, rows, tiles per row tile)}"""
    out = {}
    for b, (n, c) in enumerate(zip(new, cached)):
        for h in range(kv_heads):
            if kind == kvattn.FORWARD:
                rows = n * group
                for r in range(0, rows, row_tile):
                    m = min(row_tile, rows - r)
                    ends = []
                    for q in range(0, row_tile, TILE):
                        last = min(rows, r + q + TILE) - 1
                        keys = c + (n if tree else last // group + 1)
                        ends.append(-(-keys // TILE) if m > q else 0)
                    out[b, h, r, 0] = (0, max(ends)), m, ends
            else:
                w = min(n, window)
                chunks = -(-(w * group) // TILE)
                for key in range(0, max(c + n, 1), row_tile):
                    first = max(0, key - c - (n - w)) * group // TILE
                    out[b, h, n - w, key] = (min(first, chunks),
                                             chunks), w * group, None
    return out


def check_key_runs(segs, info, new, cached, group, kv_heads, window, tok0):
    """Weights of few rows: each segment is a run of key pairs."""
    assert info.merges == info.parts == info.workspace_bytes == 0
    runs = {}
    for s in segs:
        t0_, n, c, b, h, first, a, z, part, pairs, _, rows, key0, fill = (
            int(x) for x in s[:14])
        w = min(n, window)
        assert (t0_, n, c) == (tok0[b], new[b], cached[b])
        assert (first, rows, part) == (n - w, w * group, -1)
        assert (a, z) == (0, -(-rows // TILE)) and z <= 1 and pairs >= 1
        assert fill == (key0 + 256 * pairs >= n + c)
        runs.setdefault((b, h), []).append((key0, key0 + 256 * pairs))
    assert set(runs) == {(b, h) for b in range(len(new))
                         for h in range(kv_heads)}
    for (b, h), r in runs.items():
        r.sort()
        assert r[0][0] == 0
        assert all(x[1] == y[0] for x, y in zip(r, r[1:]))
        keys = new[b] + cached[b]
        assert r[-1][1] >= keys and r[-1][0] < max(keys, 1)


CASES = [
    ([1], [0]), ([1], [1000]), ([1] * 64, [6000 + 31 * i for i in range(64)]),
    ([16384], [0]), ([64] * 8, [4096] * 8), ([5, 0, 300, 1, 129], [0] * 5),
    ([0, 0], [0, 7]), ([400] * 4, [9000, 1, 0, 12345]), ([2], [200000]),
    ([], []), ([7] * 300, [3] * 300)]


@pytest.mark.parametrize("kind", [kvattn.FORWARD, kvattn.WEIGHTS])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("heads,kv_heads,dim,tree,window,sms", [
    (32, 8, 128, 0, 2 ** 31 - 1, 148), (7, 1, 64, 1, 33, 148),
    (4, 4, 128, 0, 1, 13), (1, 1, 64, 0, 200, 1)])
def test_every_unit_is_in_one_segment(kind, case, heads, kv_heads, dim, tree,
                                      window, sms):
    new, cached = CASES[case]
    group = heads // kv_heads
    info, buf = make(kind, new, cached, heads, kv_heads, dim, 16, tree,
                     window, sms)
    first, segs, merges = split(info, buf)
    assert info.tokens == sum(new) and info.ctas <= sms
    assert info.max_keys == max([a + b for a, b in zip(new, cached)] or [0])
    assert first[0] == 0 if info.ctas else True
    assert (np.diff(first) >= 0).all() and (
        info.ctas == 0 or first[-1] == info.segments)
    want = units(kind, new, cached, group, kv_heads, info.row_tile,
                 tree and kind == kvattn.FORWARD, window)
    got, parts = {}, {}
    tok0 = np.concatenate([[0], np.cumsum(new)])
    most = max(new or [0])
    if kind == kvattn.WEIGHTS and min(most, window) * group <= TILE:
        return check_key_runs(segs, info, new, cached, group, kv_heads,
                              window, tok0)
    for s in segs:
        t0_, n, c, b, h, row0, a, z, part, n0, n1, rows, key0, fill = (
            int(x) for x in s[:14])
        key = b, h, row0, key0
        (lo, hi), m, ends = want[key]
        assert (t0_, n, c, rows) == (tok0[b], new[b], cached[b], m)
        assert lo <= a <= z <= hi and (z > a or lo == hi)
        if ends is not None:
            ends = (ends + [0])[:2] if info.row_tile == 256 else ends + [0]
            assert n0 == max(a, min(ends[0], z))
            assert n1 == max(a, min(ends[1], z))
            assert max(n0, n1) == z
        else:
            assert fill == (key0 + 256 >= n + c)
        got.setdefault(key, []).append((a, z))
        parts.setdefault(key, []).append(part)
    assert set(got) == set(want)
    slots = set()
    listed = {(int(m[6]), int(m[1]), int(m[2]) if kind == 0 else None,
               int(m[7])): m for m in merges}
    for key, ranges in got.items():
        ranges.sort()
        assert ranges[0][0] == want[key][0][0]
        assert ranges[-1][1] == want[key][0][1]
        assert all(x[1] == y[0] for x, y in zip(ranges, ranges[1:]))
        p = sorted(parts[key])
        if len(p) == 1:
            assert p == [-1]
            continue
        b, h, row0, key0 = key
        m = listed.pop((b, h, row0 if kind == 0 else None, key0))
        assert p == list(range(int(m[4]), int(m[4]) + int(m[5])))
        assert int(m[0]) == tok0[b]
        assert int(m[3]) == (want[key][1] if kind == 0
                             else new[b] + cached[b])
        assert not slots & set(p)
        slots |= set(p)
    assert not listed and slots == set(range(info.parts))
    per = info.row_tile * (dim + 1 if kind == 0 else 1) * 4
    assert info.workspace_bytes == info.parts * per


def test_random_batches_balance():
    rng = random.Random(5)
    for _ in range(40):
        n = rng.randint(1, 80)
        new = [1] * n
        cached = [rng.randint(0, 20000) for _ in range(n)]
        info, buf = make(kvattn.FORWARD, new, cached)
        first, segs, _ = split(info, buf)
        per = [sum(int(s[7] - s[6]) for s in segs[first[c]:first[c + 1]])
               for c in range(info.ctas)]
        total = sum(per)
        if total > 148 * 40:
            assert info.ctas == 148
            assert max(per) <= 1.35 * total / 148


def test_short_buffer_is_left_alone():
    info, buf = make(kvattn.FORWARD, [1] * 64, [6000] * 64, capacity=100)
    assert info.ints > 100 and (buf == -7).all()


@pytest.mark.parametrize("kw,text", [
    (dict(dim=96), "head_dim"), (dict(heads=12, kv_heads=8), "multiple"),
    (dict(kv_heads=0), "multiple"), (dict(page=-1), "page size"),
    (dict(page=0), "page size"), (dict(new=[-1]), "negative"),
    (dict(cached=[-5]), "negative"), (dict(new=[1 << 30]), "2\\^30"),
    (dict(kind=2), "kind"), (dict(kind=1, window=0), "window"),
    (dict(new=[200000000], cached=[0], heads=8, kv_heads=1), "2\\^30")])
def test_refusals(kw, text):
    a = dict(kind=0, new=[4], cached=[10])
    a.update(kw)
    with pytest.raises(_lib.CascadeError, match=text) as e:
        make(a.pop("kind"), a.pop("new"), a.pop("cached"), **a)
    assert e.value.code == 1


def test_struct_layouts():
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    _lib.load().cascade_attn_struct_sizes(ctypes.byref(a), ctypes.byref(b))
    assert a.value == ctypes.sizeof(kvattn._PlanInfo)
    assert b.value == kvattn._ARGS.size


class Args:
    """cascade_attn_args_t by field names."""
    NAMES = ("dtype pages scale add plan q k v q_tok q_head k_tok k_head "
             "v_tok v_head k_pages v_pages kp_page kp_head kp_tok vp_page "
             "vp_head vp_tok table table_row mask mask_row out out_tok "
             "out_head lse lse_tok lse_head before before_seq before_head "
             "weights weights_seq weights_head width fill workspace "
             "workspace_bytes").split()

    def __init__(self, **kw):
        self.__dict__.update(dict.fromkeys(self.NAMES, 0), **kw)

    def pack(self):
        return kvattn._ARGS.pack(*(getattr(self, n) for n in self.NAMES))


def test_launches_refuse_bad_arguments():
    L = _lib.load()
    info, _ = make(kvattn.FORWARD, [4], [10])
    args = Args(scale=1.0)
    call = lambda fn, i, a: fn(ctypes.byref(i), a.pack(), None)
    assert L.cascade_attn_forward(None, None, None) == 1
    assert call(L.cascade_attn_weights, info, args) == 1       # wrong kind
    assert call(L.cascade_attn_forward, info, args) == 1       # no plan
    args.plan = 4096
    assert call(L.cascade_attn_forward, info, args) == 1       # no tensors
    args.q = args.k = args.v = 4096
    assert call(L.cascade_attn_forward, info, args) == 1       # no pages
    args.k_pages = args.v_pages = args.table = 4096
    args.q_tok = 4
    assert call(L.cascade_attn_forward, info, args) == 1       # alignment
    assert b"16-byte" in L.cascade_last_error()
    args.q_tok = 8
    for bad in (0.0, -1.0, 1e-30, 1e30, float("inf"), float("nan")):
        args.scale = bad
        assert call(L.cascade_attn_forward, info, args) == 1
        assert b"scale" in L.cascade_last_error()
    args.scale, args.dtype = 1.0, 2
    assert call(L.cascade_attn_forward, info, args) == 1
    args.dtype = 1
    assert call(L.cascade_attn_forward, info, args) == 1       # no output
    winfo, _ = make(kvattn.WEIGHTS, [4], [10])
    args.weights, args.lse, args.width = 4096, 4096, 13
    assert call(L.cascade_attn_weights, winfo, args) == 1      # 14 keys
    assert b"longest" in L.cascade_last_error()


def test_evict_refuses_bad_arguments():
    L = _lib.load()
    dims, st = (ctypes.c_int64 * 3)(2, 1, 1), (ctypes.c_int64 * 3)(9, 0, 0)

    def select(dims=dims, width=9, budget=4, recent=1, sink=1, w=4096,
               keep=4096):
        return L.cascade_kv_evict_select(w, dims, st, width, None, budget,
                                         recent, sink, keep, None)
    assert select(budget=0) == 1 and select(recent=-1) == 1
    assert select(recent=3, sink=2) == 1 and select(width=-1) == 1
    assert select(dims=(ctypes.c_int64 * 3)(-1, 1, 1)) == 1
    assert select(dims=(ctypes.c_int64 * 3)(1 << 20, 1 << 20, 1 << 20)) == 1
    assert select(w=None) == 1 and select(keep=None) == 1
    assert select(dims=(ctypes.c_int64 * 3)(0, 1, 1)) == 0    # no rows
    assert select(dims=None) == 1

    def gather(items=1, layers=1, heads=2, seq=9, dim=8, elem=2, keep=4096,
               kept=4, table=None, cols=0, page=0, pages=0, out=4096,
               ptr=4096):
        rows = np.array([[ptr, 72, 8]] * 2 * max(items, 1), np.int64)
        return L.cascade_kv_evict_gather(
            rows.ctypes.data, items, layers, heads, seq, dim, elem, keep,
            kept, table, cols, cols, 64, page, pages, out, None)
    assert gather(elem=1) == 1 and gather(heads=70000) == 1
    assert gather(layers=0) == 1 and gather(keep=None) == 1
    assert gather(out=None) == 1 and gather(ptr=0) == 1
    assert gather(table=4096, cols=1, page=0) == 1
    assert gather(items=0) == 0 and gather(kept=0) == 0


def test_evict_refuses_rows_that_32_bit_steps_would_pass():
    L = _lib.load()
    dims, st = (ctypes.c_int64 * 3)(2, 1, 1), (ctypes.c_int64 * 3)(9, 0, 0)
    for width, budget in ((2 ** 31 - 1, 9), ((1 << 30) + 1, 9),
                          (9, 2 ** 31 - 1), (9, (1 << 30) + 1)):
        assert L.cascade_kv_evict_select(4096, dims, st, width, None, budget,
                                         1, 1, 4096, None) == 1
        assert b"2^30" in L.cascade_last_error()


@pytest.mark.parametrize("layers", [(0, 1), (0, 0, 2), (1, 0), (2, 1)])
def test_evict_refuses_caches_of_different_layers(layers):
    kv = torch.zeros(1, 2, 9, 8, dtype=torch.float16)
    caches = [[(kv, kv)] * n for n in layers]
    with pytest.raises(ValueError, match="same layers"):
        kvattn.evict_kv_caches(caches, torch.zeros(len(layers), 2, 9), 4)
