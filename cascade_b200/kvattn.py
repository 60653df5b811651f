"""Operators over KV caches on the device: attention that reads a cache, the
attention weight each cached token received, and eviction by it.

They work on what cascade_b200.kvwire loads from the store and hand back what
it stores.  A server's step over stored prefixes:

    pages, found = kvwire.load_kv_pages(store, block_ids, ...)   # 16-token
    plan = kvattn.AttentionPlan(new, cached, q_heads=32, kv_heads=8,
                                head_dim=128, page_size=16)
    for layer in ...:                    # one plan serves every layer
        kv = pages[:, layer, 0], pages[:, layer, 1]
        out, lse = kvattn.prompt_attention(plan, q, k, v, kv, table)

New tokens are packed: `q` is [tokens, q heads, dim], `k` and `v` [tokens, kv
heads, dim], sequence after sequence; the lengths live in the plan.  Cached
tokens are in pages [pages, kv heads, page, dim] that an int32 `page_table`
[sequences, columns] names in order; the new tokens follow the cached ones.
An entry outside [0, pages) names no page: its tokens are never read and
count as unseen.  Query head h uses key/value head h // (q_heads //
kv_heads).  Tensors are float16 or bfloat16, head_dim 64 or 128 and
contiguous; other strides may be anything whose rows start on 16-byte
boundaries (a slice of a fused projection, a [1, heads, seq, dim] cache
permuted to [seq, heads, dim]).  Pages have q's type; load_kv_pages returns
float16, so a bfloat16 model converts what it loads.  Outputs share no memory
with inputs, except where a call says so.  Rows of `out` that belong to no
sequence are left as they were.  A value of V that is not finite leaves the
rows that see it not finite, and the rows that do not see it alone.  There are
no backward passes: tensors that require a gradient are refused while
gradients are enabled.

Work is enqueued on the current stream of the tensors' device.  A plan may be
used on any stream, and in captured graphs for as long as it is kept alive
(a replay has the lengths of the plan: the next decode step needs another);
workspaces are allocated per call, so calls on several streams and graphs
that overlap share nothing.  Waits inside the attention kernels are bounded:
results of a block whose wait ran out (which takes a broken device or library)
are NaN, and wait_timeouts() counts them.
"""
from __future__ import annotations

import array
import ctypes
import struct

from . import _lib, kvwire
from ._lib import check

FORWARD, WEIGHTS = 0, 1            # CASCADE_ATTN_*

_i32, _i64, _u64, _f32 = (ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64,
                          ctypes.c_float)
_vp, _u32, _int, _sz = (ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int,
                        ctypes.c_size_t)


class _PlanInfo(ctypes.Structure):
    """cascade_attn_plan_info_t."""
    _fields_ = [(n, _i32) for n in (
        "kind", "batch", "q_heads", "kv_heads", "head_dim", "page_size",
        "tree", "window", "sms", "ints", "ctas", "segments", "parts",
        "merges", "merge_rows", "row_tile", "max_new", "max_cached",
        "max_keys", "table_cols")] + [("tokens", _i64),
                                      ("workspace_bytes", _u64)]


_DIMS = struct.Struct("@3q")
# cascade_attn_args_t, in the order of _pack_args' arguments
_ARGS = struct.Struct("@iifi4P6q2P6qPqPqPqqPqqPqqPqqiiPQ")


_lib.register("cascade_attn_struct_sizes", None, [_vp, _vp])
_lib.register("cascade_attn_plan", _int, [_vp, _vp, _vp, _vp, _sz])
_lib.register("cascade_attn_forward", _int, [_vp, _vp, _vp])
_lib.register("cascade_attn_weights", _int, [_vp, _vp, _vp])
_lib.register("cascade_kv_evict_select", _int,
              [_vp, _vp, _vp, _i32, _vp, _i32, _i32, _i32, _vp, _vp])
_lib.register("cascade_kv_evict_gather", _int,
              [_vp, _u32, _u32, _u32, _u32, _u32, _u32, _vp, _u32, _vp, _i64,
               _i64, _i64, _u32, _u32, _vp, _vp])
_lib.register("cascade_diag_attn_timeouts", _int, [ctypes.POINTER(_u64)])


# ------------------------------------------------------------------- plans
def _host_lengths(x, name):
    import numpy as np
    if hasattr(x, "detach"):
        x = x.detach().cpu().numpy()
    a = np.asarray(x)
    if a.size == 0:
        a = a.astype(np.int64)
    if a.ndim != 1 or a.dtype.kind not in "iu":
        raise TypeError(f"{name} must be a 1-D sequence of integers")
    if a.size and (int(a.min()) < 0 or int(a.max()) > 1 << 30):
        raise ValueError(f"{name} must be in [0, 2**30]")
    return np.ascontiguousarray(a, dtype=np.int32)


def _cuda_device(device):
    import torch
    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError("the attention operators run on CUDA devices only")
    return d if d.index is not None else torch.device(
        "cuda", torch.cuda.current_device())


class _Plan:
    """The division of one batch among the SMs, made once on the host from
    its lengths and used by every layer's call."""

    def __init__(self, kind, new_lengths, cached_lengths, q_heads, kv_heads,
                 head_dim, page_size, device, tree=False, window=1):
        import numpy as np
        import torch
        new = _host_lengths(new_lengths, "new_lengths")
        cached = (np.zeros_like(new) if cached_lengths is None
                  else _host_lengths(cached_lengths, "cached_lengths"))
        if cached.size != new.size:
            raise ValueError("one cached length per sequence: "
                             f"{cached.size} for {new.size}")
        page_size = page_size or 0
        for name, n in (("q_heads", q_heads), ("kv_heads", kv_heads),
                        ("head_dim", head_dim), ("page_size", page_size)):
            if not 0 <= n < 1 << 31:
                raise ValueError(f"{name} must be in [0, 2**31); got {n}")
        self.device = _cuda_device(device)
        info = _PlanInfo(
            kind=kind, batch=new.size, q_heads=q_heads, kv_heads=kv_heads,
            head_dim=head_dim, page_size=page_size, tree=int(tree),
            window=window)
        with torch.cuda.device(self.device):
            buf = np.empty(4096, np.int32)
            for _ in range(2):
                check(_lib.load().cascade_attn_plan(
                    ctypes.byref(info), new.ctypes.data, cached.ctypes.data,
                    buf.ctypes.data, buf.size))
                if info.ints <= buf.size:
                    break
                buf = np.empty(info.ints, np.int32)
            # a blocking copy: the plan is ready for every stream
            self._buf = torch.from_numpy(buf[:info.ints].copy()).to(
                self.device)
            # new_empty of a tensor takes less time than torch.empty
            self._f32 = torch.empty(0, device=self.device,
                                    dtype=torch.float32)
        self._stream = _raw_stream(self.device.index)
        self._info = info
        self._ref = ctypes.byref(info)
        self.batch, self.tokens = info.batch, info.tokens
        self.q_heads, self.kv_heads = info.q_heads, info.kv_heads
        self.head_dim, self.page_size = info.head_dim, info.page_size
        self.max_new, self.max_cached = info.max_new, info.max_cached
        self.max_keys, self.tree = info.max_keys, bool(info.tree)
        self._heads = q_heads, kv_heads, head_dim
        self._ptr, self._lib = self._buf.data_ptr(), _lib.load()


class AttentionPlan(_Plan):
    """Plan of prompt_attention (or, with tree=True, tree_attention) for a
    batch of sequences with `new_lengths` new tokens each behind
    `cached_lengths` cached ones (host integers; None: none cached)."""

    def __init__(self, new_lengths, cached_lengths=None, *, q_heads,
                 kv_heads, head_dim, page_size=None, tree=False,
                 device="cuda"):
        super().__init__(FORWARD, new_lengths, cached_lengths, q_heads,
                         kv_heads, head_dim, page_size, device, tree=tree)


class WeightsPlan(_Plan):
    """Plan of attention_weights.  `window`: how many of each sequence's
    last new tokens count (None: all)."""

    def __init__(self, new_lengths, cached_lengths=None, *, q_heads,
                 kv_heads, head_dim, page_size=None, window=None,
                 device="cuda"):
        if window is None:
            window = (1 << 31) - 1
        if not 0 < window < 1 << 31:
            raise ValueError("window must be above 0")
        super().__init__(WEIGHTS, new_lengths, cached_lengths, q_heads,
                         kv_heads, head_dim, page_size, device,
                         window=window)


# ------------------------------------------------------------------ checks
def _dtype_code(q):
    import torch
    if q.dtype is torch.float16:
        return 0
    if q.dtype is torch.bfloat16:
        return 1
    raise TypeError(f"q must be float16 or bfloat16, not {q.dtype}")


def _strides(t):
    """Element strides with 0 for dimensions of one element, whose stride
    torch leaves arbitrary."""
    return tuple(0 if n == 1 else s for n, s in zip(t.shape, t.stride()))


def _rows(name, t, shape, dtype, device):
    """(address, strides) of a tensor of 16-bit rows."""
    p, st = t.data_ptr(), t.stride()
    if (t.shape == shape and t.dtype is dtype and t.device == device
            and st[-1] == 1 and not (p | st[0] * 2 | st[1] * 2
                                     | st[-2] * 2) & 15):
        return p, st
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}; got "
                         f"{tuple(t.shape)}")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} on {device}; got {t.dtype} "
                         f"on {t.device}")
    if st[-1] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    st = _strides(t)
    if p % 16 or any(s % 8 for s in st[:-1]):
        raise ValueError(f"{name}: rows must start on 16-byte boundaries")
    return p, st


try:                               # the plain calls, without Python objects
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
    from torch._C import _cuda_getDevice as _current_device
except ImportError:                # pragma: no cover - other torch versions
    def _raw_stream(index):
        import torch
        return torch.cuda.current_stream(index).cuda_stream

    def _current_device():
        import torch
        return torch.cuda.current_device()


def _launch(device, fn, *args):
    """fn(*args, current stream of `device`), with that device current."""
    if _current_device() == device.index:
        check(fn(*args, _raw_stream(device.index)))
        return
    import torch
    with torch.cuda.device(device):
        check(fn(*args, _raw_stream(device.index)))


def _no_grad(*tensors):
    import torch
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("operators over KV caches have no "
                                   "backward pass: call them under "
                                   "torch.no_grad()")


def _writable(name, t):
    if any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} must not be an expanded tensor")


def _scale(scale, dim):
    if scale is None:
        return dim ** -0.5
    if not 2.0 ** -64 <= scale <= 2.0 ** 64:
        raise ValueError("scale must be in [2**-64, 2**64]")
    return scale


def _table(page_table, batch, cols, dev):
    import torch
    if (page_table.dim() != 2 or page_table.shape[0] != batch
            or page_table.shape[1] < cols):
        raise ValueError(f"page_table must be [{batch}, >= {cols}]; got "
                         f"{tuple(page_table.shape)}")
    if page_table.dtype is not torch.int32 or page_table.device != dev:
        raise ValueError(f"page_table must be int32 on {dev}")
    st = page_table.stride()
    if page_table.shape[1] > 1 and st[1] != 1:
        raise ValueError("page_table: rows must be contiguous")
    return page_table.data_ptr(), st[0] if batch > 1 else 0


_NO_KV = (0,) * 4


def _call(plan, kind, fn, q, k, v, k_pages, v_pages, page_table, scale, add,
          mask, out, lse, before, weights):
    """Checks the arguments that both kinds of call share and runs fn on the
    current stream of the plan's device.  mask: (address, stride); out, lse,
    before: (address, strides); weights: (address, strides, width, fill)."""
    import torch
    if plan._info.kind != kind:
        raise ValueError("the plan is of the other kind: AttentionPlan for "
                         "attention, WeightsPlan for attention_weights")
    dev, dt = plan.device, q.dtype
    rows, (H, G, D) = q.shape[0], plan._heads
    if rows < plan.tokens:
        raise ValueError(f"q must be [>= {plan.tokens} tokens, {H}, {D}]; "
                         f"got {tuple(q.shape)}")
    code = _dtype_code(q)
    qp, qs = _rows("q", q, (rows, H, D), dt, dev)
    kp, ks = _rows("k", k, (rows, G, D), dt, dev)
    vp, vs = (0, _NO_KV) if v is None else _rows("v", v, (rows, G, D), dt,
                                                 dev)
    P = pkp = pvp = tp = trow = 0
    pks = pvs = _NO_KV
    if plan.max_cached:
        if k_pages is None or page_table is None:
            raise ValueError("the plan has cached tokens: pages and "
                             "page_table are needed")
        P = k_pages.shape[0]
        shape = (P, G, plan.page_size, D)
        pkp, pks = _rows("k_pages", k_pages, shape, dt, dev)
        if v is not None:
            if v_pages is None:
                raise ValueError("pages is a pair (k_pages, v_pages)")
            pvp, pvs = _rows("v_pages", v_pages, shape, dt, dev)
        tp, trow = _table(page_table, plan.batch, plan._info.table_cols, dev)
    scale = _scale(scale, D)
    if _raw_stream(dev.index) != plan._stream:
        # the plan's memory must not be handed out while this call reads
        plan._buf.record_stream(torch.cuda.current_stream(dev))
    size = plan._info.workspace_bytes
    # freed on return: the allocator hands it out again only to work
    # ordered behind this call on the same stream
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    args = _ARGS.pack(
        code, P, scale, add, plan._ptr, qp, kp, vp, qs[0], qs[1], ks[0],
        ks[1], vs[0], vs[1], pkp, pvp, pks[0], pks[1], pks[2], pvs[0],
        pvs[1], pvs[2], tp, trow, mask[0], mask[1], out[0], out[1][0],
        out[1][1], lse[0], lse[1][0], lse[1][1], before[0], before[1][0],
        before[1][1], weights[0], weights[1][0], weights[1][1],
        weights[2], weights[3], ws.data_ptr() if size else 0, size)
    _launch(dev, fn, plan._ref, args)


_NONE = (0, (0, 0))


# --------------------------------------------------------------- attention
def _forward(plan, q, k, v, mask, pages, page_table, scale, out, lse):
    import torch
    k_pages, v_pages = pages if pages is not None else (None, None)
    _no_grad(q, k, v, k_pages, v_pages)
    if q.dim() != 3:
        raise ValueError("q must be [tokens, q heads, dim]; got "
                         f"{tuple(q.shape)}")
    dev, rows = plan.device, q.shape[0]
    H, _, D = plan._heads
    mp = (0, 0)
    if mask is not None:
        if (mask.dim() != 2 or mask.shape[0] != rows
                or mask.shape[1] < plan.max_new):
            raise ValueError(f"mask must be [{rows}, >= {plan.max_new}]; "
                             f"got {tuple(mask.shape)}")
        if (mask.dtype is not torch.bool and mask.dtype is not torch.uint8
                ) or mask.device != dev:
            raise ValueError(f"mask must be bool or uint8 on {dev}")
        if mask.shape[1] > 1 and mask.stride(1) != 1:
            raise ValueError("mask: rows must be contiguous")
        mp = mask.data_ptr(), mask.stride(0)
    if out is None:
        # (_call refuses a q of another shape or device)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        op = out.data_ptr(), (H * D, D)
    else:
        _writable("out", out)
        op = _rows("out", out, (rows, H, D), q.dtype, dev)
    if lse is None:
        lse = plan._f32.new_empty((rows, H))
        lp = lse.data_ptr(), (H, 1)
    else:
        _writable("lse", lse)
        if (tuple(lse.shape) != (rows, H) or lse.dtype != torch.float32
                or lse.device != dev):
            raise ValueError(f"lse must be float32 {(rows, H)} on {dev}")
        lp = lse.data_ptr(), _strides(lse)
    _call(plan, FORWARD, plan._lib.cascade_attn_forward, q, k, v, k_pages,
          v_pages, page_table, scale, 0, mp, op, lp, _NONE, (0, (0, 0), 0, 0))
    return out, lse


def prompt_attention(plan, q, k, v, pages=None, page_table=None, *,
                     scale=None, out=None, lse=None):
    """Causal attention of packed new tokens: each sees its sequence's cached
    tokens and the new ones up to itself.  Whole prompts, the rest of a
    prompt whose prefix came from the store, and single tokens of a decode
    step are all this call; they differ in the plan's lengths only.

    q [tokens, q heads, dim], k and v [tokens, kv heads, dim]; pages =
    (k_pages, v_pages) and page_table where the plan has cached tokens;
    scale defaults to 1 / sqrt(dim).  Returns (out, lse): out as q, lse
    float32 [tokens, q heads], the natural log of the sum of exp(score)."""
    if plan.tree:
        raise ValueError("the plan is for trees: use tree_attention")
    return _forward(plan, q, k, v, None, pages, page_table, scale, out, lse)


def tree_attention(plan, q, k, v, mask, pages=None, page_table=None, *,
                   scale=None, out=None, lse=None):
    """Attention of drafted tokens, which are not in the cache yet: each sees
    its sequence's cached tokens and the drafts its mask row names.  mask
    [tokens, >= longest tree] bool: mask[t, j] says that packed token t sees
    draft j of its own sequence (itself only where the mask says so).  A
    token that sees nothing at all gets zeros and lse -inf.  The plan is made
    with tree=True; otherwise as prompt_attention."""
    if not plan.tree:
        raise ValueError("the plan is causal: make it with tree=True")
    if mask is None:
        raise ValueError("tree_attention needs a mask")
    return _forward(plan, q, k, v, mask, pages, page_table, scale, out, lse)


def _weight_rows(name, t, plan):
    import torch
    if (t.dim() != 3 or t.shape[0] != plan.batch
            or t.shape[1] != plan.kv_heads or t.shape[2] < plan.max_keys):
        raise ValueError(
            f"{name} must be [{plan.batch}, {plan.kv_heads}, >= "
            f"{plan.max_keys}]; got {tuple(t.shape)}")
    if t.dtype is not torch.float32 or t.device != plan.device:
        raise ValueError(f"{name} must be float32 on {plan.device}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return t.data_ptr(), t.stride()


def attention_weights(plan, q, k, lse, k_pages=None, page_table=None, *,
                      scale=None, add_to=None, out=None):
    """The attention weight that every token received: out[b, kv head, j] =
    add_to + the sum of exp(score - lse) over the query heads of the group
    and the last `window` new tokens of sequence b that see token j
    (causally).  lse is prompt_attention's, for the same tokens and scale.

    add_to and out are float32 [sequences, kv heads, width >= longest
    sequence] with contiguous rows; out may be add_to itself.  Returns out;
    without one, a new tensor whose positions behind a sequence's end hold
    add_to's values (or 0).  In a given out those are left as they were."""
    import torch
    _no_grad(q, k, lse, k_pages, add_to)
    if q.dim() != 3:
        raise ValueError("q must be [tokens, q heads, dim]; got "
                         f"{tuple(q.shape)}")
    dev = plan.device
    if (lse.dim() != 2 or lse.shape[0] != q.shape[0]
            or lse.shape[1] != plan.q_heads
            or lse.dtype is not torch.float32 or lse.device != dev):
        raise ValueError("lse must be float32 "
                         f"{(q.shape[0], plan.q_heads)} on {dev}")
    lp = lse.data_ptr(), lse.stride()
    bp, add, fill = _NONE, 0, 0
    if add_to is not None:
        bp, add = _weight_rows("add_to", add_to, plan), 1
    if out is None:
        width = plan.max_keys if add_to is None else add_to.shape[2]
        out = plan._f32.new_empty((plan.batch, plan.kv_heads, width))
        wp, fill = (out.data_ptr(), out.stride()), 1
    else:
        _writable("out", out)
        wp = _weight_rows("out", out, plan)
        width = out.shape[2] if add_to is None else min(out.shape[2],
                                                        add_to.shape[2])
    _call(plan, WEIGHTS, plan._lib.cascade_attn_weights, q, k, None, k_pages,
          None, page_table, scale, add, (0, 0), _NONE, lp, bp,
          (wp[0], wp[1], width, fill))
    return out


# ---------------------------------------------------------------- eviction
def select_kept(weights, budget, recent=0, sink=0, lengths=None):
    """The tokens to keep: weights is float32 [sequences, ..., tokens] (up to
    three leading dimensions, contiguous rows).  Each row keeps its first
    `sink` and last `recent` tokens and those of the largest weights, ties to
    the lowest position, `budget` in all; NaN ranks with minus infinity.
    lengths (int32 CUDA [sequences], clamped to the row) ends the rows of a
    sequence early.  Returns int32 [sequences, ..., budget], ascending; a row
    of fewer tokens than budget keeps all and ends in -1."""
    import torch
    _no_grad(weights)
    if weights.dtype != torch.float32 or not weights.is_cuda:
        raise ValueError("weights must be a float32 CUDA tensor")
    if not 2 <= weights.dim() <= 4:
        raise ValueError("weights has 1 to 3 dimensions before the tokens; "
                         f"got shape {tuple(weights.shape)}")
    lead = tuple(weights.shape[:-1])
    if lengths is not None and (
            lengths.dtype != torch.int32 or lengths.device != weights.device
            or tuple(lengths.shape) != (lead[0],)
            or not lengths.is_contiguous()):
        raise ValueError(f"lengths must be int32 [{lead[0]}] on "
                         f"{weights.device}")
    return _select(weights, lead, weights.shape[-1], weights.device, budget,
                   recent, sink, lengths)


def _select(weights, lead, width, dev, budget, recent, sink, lengths=None):
    """select_kept for float32 weights of shape (*lead, width) on dev."""
    import torch
    st = weights.stride()
    if width > 1 and st[-1] != 1:
        raise ValueError("weights: rows must be contiguous")
    if budget < 1 or recent < 0 or sink < 0 or recent + sink > budget:
        raise ValueError("budget must be above 0 and at least recent + sink "
                         f"(got {budget}, {recent}, {sink})")
    if max(budget, width) > 1 << 30:
        raise ValueError("rows have at most 2**30 tokens")
    keep = weights.new_empty(lead + (budget,), dtype=torch.int32)
    pad = 3 - len(lead)
    _launch(dev, _lib.load().cascade_kv_evict_select, weights.data_ptr(),
            _DIMS.pack(*lead, *(1,) * pad),
            _DIMS.pack(*st[:-1], *(0,) * pad), width,
            lengths.data_ptr() if lengths is not None else None, budget,
            recent, sink, keep.data_ptr())
    return keep


def evict_kv_caches(caches, weights, budget, recent=0, sink=0):
    """Shortens n KV caches of one shape (as kvwire.serialize_kv_caches
    takes them) to `budget` tokens per head by select_kept's rule.  weights:
    float32 [n, layers, kv heads, seq], or [n, kv heads, seq] for one choice
    that all layers share.

    Returns (kv, keep): kv [n, layers, 2, kv heads, kept, dim] in the caches'
    dtype (kept = min(budget, seq)) and the positions, int32 [n, (layers,)
    kv heads, kept].  cache_views(kv) gives the caches back as tuples."""
    import torch
    n = len(caches)
    if n == 0:
        raise ValueError("no caches to evict from")
    per = [kvwire.extract_kv_pairs(c) for c in caches]
    L = len(per[0])
    if any(len(pairs) != L for pairs in per):
        raise ValueError("every cache must have the same layers")
    if L == 0:
        raise ValueError("a KV cache needs at least one layer")
    tensors = [t for pairs in per for kv in pairs for t in kv]
    _no_grad(weights, *tensors)
    t0 = tensors[0]
    if t0.dim() not in (3, 4):
        raise ValueError("KV tensors are [1, heads, seq, dim]; got "
                         f"{tuple(t0.shape)}")
    (H, S, D), dev, dt = t0.shape[-3:], t0.device, t0.dtype
    lead = (n, L, H) if weights.dim() == 4 else (n, H)
    if tuple(weights.shape) != lead + (S,) or weights.device != dev:
        raise ValueError(f"weights must be {lead + (S,)} on {dev}; got "
                         f"{tuple(weights.shape)} on {weights.device}")
    if budget >= S and 0 <= recent and 0 <= sink and \
            recent + sink <= budget:
        recent, sink = min(recent, S), 0         # everything is kept
        budget = max(S, 1)
    if weights.dtype is not torch.float32 or dev.type != "cuda":
        raise ValueError("weights must be a float32 CUDA tensor")
    # the choice is made while the host looks the tensors over
    keep = _select(weights, lead, S, dev, budget, recent, sink)
    desc = _descriptors(tensors, (H, S, D), dev, dt)
    kept = min(budget, S)
    if kept < budget:
        keep = keep[..., :kept]
    kv = t0.new_empty((n, L, 2, H, kept, D))
    _launch(dev, _lib.load().cascade_kv_evict_gather, desc.buffer_info()[0],
            n * L, L if len(lead) == 2 else 1, H, S, D, dt.itemsize,
            keep.data_ptr(), kept, None, 0, 0, 0, 0, 0, kv.data_ptr())
    return kv, keep


def _descriptors(tensors, shape, dev, dt):
    """Host cascade_kv_tensor_t rows, as an array, of [1, heads, seq, dim] or
    [heads, seq, dim] tensors, all of `shape` on `dev`."""
    import torch
    if dt.itemsize not in (2, 4):
        raise ValueError("KV tensors are CUDA tensors of 2- or 4-byte values")
    H, S, D = shape
    n, one, T = len(tensors), (1, H, S, D), torch.Tensor
    # whole lists at a time: 0.4 us a tensor, one by one 0.65
    sizes = [t.shape for t in tensors]
    if (sizes.count(one) + sizes.count(shape) != n
            or [t.dtype for t in tensors].count(dt) != n
            or list(map(T.get_device, tensors)).count(dev.index) != n):
        raise ValueError("every K and V must have one shape ([1,] heads, "
                         "seq, dim), dtype and device")
    rows = array.array("q", bytes(24 * n))
    rows[0::3] = array.array("q", map(T.data_ptr, tensors))
    strides = list(map(T.stride, tensors))
    if strides.count(strides[0]) == n:          # the usual case
        strides = strides[:1]
    for i, st in enumerate(strides):
        if st[-1] != 1 and D > 1:
            raise ValueError("head_dim must be contiguous (stride 1)")
        rows[3 * i + 1] = st[-3] if H > 1 else 0
        rows[3 * i + 2] = st[-2] if S > 1 else 0
    if len(strides) < n:
        rows[1::3] = rows[1:2] * n
        rows[2::3] = rows[2:3] * n
    return rows


def cache_views(kv):
    """evict_kv_caches' kv as a list of caches: tuples of (K, V) per layer,
    [1, kv heads, kept, dim] each."""
    return [tuple((l[0].unsqueeze(0), l[1].unsqueeze(0)) for l in c)
            for c in kv]


def evict_pages(k_pages, v_pages, page_table, lengths, weights, budget,
                recent=0, sink=0):
    """The same for one layer of a batch in pages: sequence b's tokens are
    the first lengths[b] (int32 CUDA [sequences]) of the pages that its row
    of page_table names, and no more than weights, float32 [sequences, kv
    heads, tokens], has.

    Returns (k, v, keep): [sequences, kv heads, budget, dim] each and the
    positions, int32 [sequences, kv heads, budget].  A sequence of fewer
    tokens keeps them all; its rows behind them are zeros and -1."""
    import torch
    _no_grad(k_pages, v_pages)
    dev, dt = k_pages.device, k_pages.dtype
    if not k_pages.is_cuda or dt.itemsize not in (2, 4):
        raise ValueError("pages must be CUDA tensors of 2- or 4-byte values")
    if (k_pages.dim() != 4 or v_pages.shape != k_pages.shape
            or v_pages.dtype != dt or v_pages.device != dev):
        raise ValueError("k_pages and v_pages must be [pages, heads, page, "
                         "dim] of one shape, dtype and device")
    P, H, page, D = k_pages.shape
    B = page_table.shape[0] if page_table.dim() else 0
    if (weights.dim() != 3 or tuple(weights.shape[:2]) != (B, H)
            or weights.device != dev):
        raise ValueError(f"weights must be [{B}, {H}, tokens] on {dev}")
    if page < 1:
        raise ValueError("pages hold at least one token")
    ks, vs = _strides(k_pages), _strides(v_pages)
    if ks[0] != vs[0]:
        raise ValueError("k_pages and v_pages must have one page stride")
    if D > 1 and not ks[3] == vs[3] == 1:
        raise ValueError("head_dim must be contiguous (stride 1)")
    table, table_row = _table(page_table, B, 0, dev)
    keep = select_kept(weights, budget, recent, sink, lengths)
    kv = k_pages.new_empty((B, 2, H, budget, D))
    if kv.numel():
        desc = struct.pack("@6q", k_pages.data_ptr(), ks[1], ks[2],
                           v_pages.data_ptr(), vs[1], vs[2])
        _launch(dev, _lib.load().cascade_kv_evict_gather, desc * B, B, 1, H,
                0, D, dt.itemsize, keep.data_ptr(), budget, table, table_row,
                page_table.shape[1], ks[0], page, P, kv.data_ptr())
    return (*kv.unbind(1), keep)


def wait_timeouts() -> int:
    """Waits inside attention kernels that gave up on the current device
    (0 unless something is broken); the results of their blocks are NaN.
    Synchronises."""
    n = _u64(0)
    check(_lib.load().cascade_diag_attn_timeouts(ctypes.byref(n)))
    return n.value
