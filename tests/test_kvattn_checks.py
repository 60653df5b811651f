"""What the operators over KV caches refuse before anything is launched, on a
machine without a GPU."""
import ctypes
import os

import pytest
import torch

from cascade_b200 import _lib, kvattn
from test_attn_plan import Args, make

CPU = torch.device("cpu")


@pytest.mark.parametrize("t", [
    torch.ones(1, dtype=torch.float16).expand(6, 4, 64),
    torch.ones(6, 4, 8, dtype=torch.float16)[..., :1].expand(6, 4, 64),
    torch.ones(64, 4, 6, dtype=torch.float16).permute(2, 1, 0),
    torch.ones(6, 4, 128, dtype=torch.float16)[..., ::2]])
def test_rows_must_be_contiguous(t):
    # a row is read as 64 values in a row: an expanded one has only one
    with pytest.raises(ValueError, match="contiguous"):
        kvattn._rows("q", t, (6, 4, 64), torch.float16, CPU)


@pytest.mark.parametrize("t,strides", [
    (torch.ones(6, 4, 64, dtype=torch.float16), (256, 64, 1)),
    (torch.ones(1, 1, 64, dtype=torch.float16).expand(6, 4, 64), (0, 0, 1)),
    (torch.ones(6, 4, 72, dtype=torch.float16)[..., :64], (288, 72, 1)),
    (torch.ones(0, 4, 64, dtype=torch.float16), (256, 64, 1))])
def test_other_strides_are_taken(t, strides):
    got = kvattn._rows("q", t, tuple(t.shape), torch.float16, CPU)
    assert got == (t.data_ptr(), strides)


@pytest.mark.parametrize("width,fill", [(0, 0), (0, 1), (9, 0)])
def test_weights_without_keys_write_nothing(width, fill):
    # an empty tensor has no address
    info, _ = make(kvattn.WEIGHTS, [0, 0], [0, 0])
    args = Args(scale=1.0, plan=4096, width=width, fill=fill,
                weights=4096 if width else 0)
    assert _lib.load().cascade_attn_weights(
        ctypes.byref(info), args.pack(), None) == 0


@pytest.mark.parametrize("kind", [kvattn.FORWARD, kvattn.WEIGHTS])
def test_no_pages_at_all_are_taken(kind):
    # every table entry is then outside [0, 0); the call goes on to what it
    # looks at next
    info, _ = make(kind, [4], [10])
    args = Args(scale=1.0, plan=4096, q=4096, k=4096, v=4096, table=4096)
    call = (_lib.load().cascade_attn_forward if kind == kvattn.FORWARD
            else _lib.load().cascade_attn_weights)
    assert call(ctypes.byref(info), args.pack(), None) == 1
    assert b"pages" not in _lib.load().cascade_last_error()
    args.pages = 1
    assert call(ctypes.byref(info), args.pack(), None) == 1
    assert b"pages" in _lib.load().cascade_last_error()


@pytest.mark.parametrize("kw", [
    dict(page_size=2 ** 32 + 16), dict(page_size=-16),
    dict(q_heads=2 ** 32 + 4), dict(kv_heads=2 ** 32 + 2),
    dict(head_dim=2 ** 32 + 64)])
@pytest.mark.parametrize("cls", [kvattn.AttentionPlan, kvattn.WeightsPlan])
def test_plan_sizes_beyond_32_bits(cls, kw):
    # the C fields have 32 bits: 2^32 + 16 must not become 16
    a = dict(q_heads=4, kv_heads=2, head_dim=64, page_size=16,
             device="cuda:0")
    a.update(kw)
    with pytest.raises(ValueError, match=next(iter(kw))):
        cls([1], [1], **a)


@pytest.mark.parametrize("name", ["attn.cu", "attn_weights.cu"])
def test_tensor_memory_is_taken_behind_the_wait(name):
    # A block launched early that holds all of an SM's tensor memory while it
    # waits for the kernel before, and a block of that kernel which has yet
    # to get some, would wait for each other.  No test can run that, so the
    # order is read from the source: wait, take, let the next start.
    path = os.path.join(os.path.dirname(kvattn.__file__), "csrc", name)
    with open(path) as f:
        text = f.read()
    assert text.count("tc_alloc(") == 1
    at = text.index("tc_alloc(")
    start = text.rindex("__global__", 0, at)
    wait = text.index("wait_for_previous();", start)
    sync = text.index("__syncthreads();", at)
    assert wait < at < sync < text.index("let_next_start();", start)


@pytest.mark.parametrize("name", ["attn.cu", "attn.cuh", "attn_weights.cu"])
def test_waits_are_counted_not_timed(name):
    # a process that another one keeps from the GPU for seconds has waited
    # for nothing: no wait may give up by the clock
    path = os.path.join(os.path.dirname(kvattn.__file__), "csrc", name)
    with open(path) as f:
        text = f.read()
    assert not any(x in text for x in ("globaltimer", "clock64", "clock("))
